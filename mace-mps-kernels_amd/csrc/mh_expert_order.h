// mh_expert_order.h — the places of rows sorted by expert, prepended with mh_device.h.
//
// A = T k assignments, experts[i] in [0, E) (anything else: dropped), i = t k + j the j-th expert of node t.  The places of
// the kept ones are their positions in a stable sort by expert; the dropped ones follow after the last group, also in
// order.  rows[place] = i (-1 where the assignment was dropped), place[i] (-1: dropped), offsets[e] the first place of e.
#pragma once

#define EX_MAX 1024                 // experts (LDS tables)
#define EX_CHUNK 1024               // assignments a workgroup ranks at once (16 waves)

__device__ __forceinline__ int ex_key(const void* experts, int wide, int i, int E) {
    const long long v = wide ? static_cast<const long long*>(experts)[i] : (long long)static_cast<const int*>(experts)[i];
    return v >= 0 && v < E ? (int)v : E;
}

// hist[b][e]: assignments of expert e among block b's `per` ones (e = E: dropped)
extern "C" __global__ __launch_bounds__(1024) void expert_hist(const void* __restrict__ experts, int wide, int A, int E, int per,
                                                                int* __restrict__ hist) {
    __shared__ int h[EX_MAX + 1];
    for (int e = threadIdx.x; e <= E; e += 1024) h[e] = 0;
    __syncthreads();
    const int hi = min(A, (int)(blockIdx.x + 1) * per);
    for (int i = blockIdx.x * per + threadIdx.x; i < hi; i += 1024) atomicAdd(&h[ex_key(experts, wide, i, E)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= E; e += 1024) hist[(long long)blockIdx.x * (E + 1) + e] = h[e];
}

// The places, block b for its `per` assignments (a multiple of EX_CHUNK): where each expert's run starts for this block
// follows from the blocks' histograms (nb of them; one block counts for itself), then chunks of 1024 are ranked: within a
// wave by the lanes that hold the same key, found with one ballot per bit of it, across waves by counts in LDS.  Bound by
// latency, not by its 12 bytes an assignment: 160 of them 3.7 us in one workgroup, 131,072 with 128 experts 13.6 us in 32 (and
// 4.9 for their histograms), a chunk of 1,024 about 2.4 us.
extern "C" __global__ __launch_bounds__(1024) void expert_place(const void* __restrict__ experts, int wide, int A, int E, int per,
                                                                 const int* __restrict__ hist, int* __restrict__ offsets,
                                                                 int* __restrict__ rows, int* __restrict__ place) {
    __shared__ int run[EX_MAX + 1], wsum[16];
    __shared__ unsigned short cnt[16][EX_MAX + 1];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, nb = gridDim.x, b = blockIdx.x;
    for (int k = t; k < 16 * (EX_MAX + 1); k += 1024) (&cnt[0][0])[k] = 0;
    if (t <= E && t <= EX_MAX) run[t] = 0;
    if (t == 0) run[E] = 0;
    __syncthreads();
    // all of expert t's assignments, and those of the blocks before this one (thread t; E = 1024 leaves key E to thread 0)
    int before = 0, all = 0;
    if (nb == 1) {
        for (int i = t; i < A; i += 1024) atomicAdd(&run[ex_key(experts, wide, i, E)], 1);
        __syncthreads();
        all = t < E ? run[t] : 0;
        __syncthreads();
    } else if (t < E) {
#pragma unroll 8
        for (int k = 0; k < nb; ++k) {
            const int c = hist[(long long)k * (E + 1) + t];
            before += k < b ? c : 0;
            all += c;
        }
    }
    int total;
    const int start = mh_block_excl_scan<int, 16>(all, total, wsum);
    if (t < E) run[t] = start + before;
    if (t == 0) {
        int d = 0;                                       // dropped ones of the blocks before
        for (int k = 0; k < (nb == 1 ? 0 : b); ++k) d += hist[(long long)k * (E + 1) + E];
        run[E] = total + d;
    }
    if (b == 0) {
        if (t < E) offsets[t] = start;
        if (t == 0) offsets[E] = total;
    }
    __syncthreads();
    const int hi = min(A, (b + 1) * per);
    for (int base = b * per; base < hi; base += EX_CHUNK) {
        const int i = base + t;
        const bool in = i < hi;
        const int e = in ? ex_key(experts, wide, i, E) : E + 1;
        unsigned long long same = __ballot(in);
        for (int bit = 0; (E + 1) >> bit; ++bit) {
            const unsigned long long set = __ballot((e >> bit) & 1);
            same &= (e >> bit) & 1 ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (in && rank == 0) cnt[wave][e] = (unsigned short)__popcll(same);
        __syncthreads();
        if (in) {
            int p = run[e] + rank;
            for (int w = 0; w < wave; ++w) p += cnt[w][e];
            rows[p] = e < E ? i : -1;
            place[i] = e < E ? p : -1;
        }
        __syncthreads();
        for (int k = t; k <= E; k += 1024) {
            int c = 0;
            for (int w = 0; w < 16; ++w) {
                c += cnt[w][k];
                cnt[w][k] = 0;
            }
            run[k] += c;
        }
        __syncthreads();
    }
}
