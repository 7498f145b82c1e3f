// mh_halves.h — float32 matrix products as three float16 ones, prepended with mh_device.h and mh_matmul.h.
//
// A row (or column) of values times a power of two s that brings its largest to [2^14, 2^15) is, value by value, hi + lo with
// hi and lo float16: hi the nearest, lo the nearest to what is left, together off by at most 2^-24 of the value, or 2^-40 of
// the row's largest where that is more.  a b = (hi_a + lo_a)(hi_b + lo_b) / (s_a s_b), where lo_a lo_b is below 2^-24 of
// |a b| and left out: three products on the matrix cores where three bf16 parts need six, at the price of a pass that writes
// the halves (s must not change along the contraction, so one s per row of an operand that is contiguous along it, one per
// column and group of an operand whose rows are contracted).  Both forms keep the halves next to each other, as matrices of
// 16-bit values whose contraction is twice as long, which the tiles of mh_matmul.h load as they are:
//   rows    [R][Kp / 32][2][32]    32 hi, their 32 lo, ...; Kp = K rounded up to 32, zeros behind K
//   columns [R][2][Cp]             a row of hi, its row of lo; Cp = C rounded up to 8
// Infinite and NaN values are hi as they are, lo 0.  Their rows and columns are marked, and what they reach is taken from the
// products hi hi alone, which give what a float32 sum gives.
#pragma once

#define HV_ODD 0x80000000u          // in a peak: the row or column holds an infinity or NaN

// exponent of s for the largest finite magnitude (its bits): 2^126 at most, beyond which float32 has no s
__device__ __forceinline__ int hv_shift(unsigned peak) {
    const int e = (int)((peak & 0x7FFFFFFFu) >> 23);
    return (peak & 0x7FFFFFFFu) ? min(14 - (e - 127), 126) : 0;
}

__device__ __forceinline__ void hv_split(float v, int shift, unsigned short& hi, unsigned short& lo) {
    const float t = __builtin_ldexpf(v, shift);
    const _Float16 h = (_Float16)t;
    const _Float16 l = (_Float16)(t - (float)h);
    hi = __builtin_bit_cast(unsigned short, h);
    lo = __builtin_isfinite(v) ? __builtin_bit_cast(unsigned short, l) : (unsigned short)0;
}

__device__ __forceinline__ void hv_split4(mh_f4 v, int4 shift, unsigned short* hi, unsigned short* lo) {
    unsigned short h[4], l[4];
    hv_split(v.x, shift.x, h[0], l[0]);
    hv_split(v.y, shift.y, h[1], l[1]);
    hv_split(v.z, shift.z, h[2], l[2]);
    hv_split(v.w, shift.w, h[3], l[3]);
    *reinterpret_cast<mh_u2*>(hi) = mh_u2{h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16};
    *reinterpret_cast<mh_u2*>(lo) = mh_u2{l[0] | (unsigned)l[1] << 16, l[2] | (unsigned)l[3] << 16};
}

// the bits of |v| where it is finite, HV_ODD where not
__device__ __forceinline__ unsigned hv_peak(float v) {
    const unsigned b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : HV_ODD;
}

// Largest of peaks, odd if any is
__device__ __forceinline__ unsigned hv_max(unsigned a, unsigned b) {
    return max(a & 0x7FFFFFFFu, b & 0x7FFFFFFFu) | ((a | b) & HV_ODD);
}

// Rows: a wave each; the second reading of a row comes from the caches.  Bound by its bytes: 20,000 rows of 1,024 in 38 us, 4.3 TB/s.
extern "C" __global__ __launch_bounds__(256) void hv_rows(const float* __restrict__ x, unsigned short* __restrict__ y,
                                                          unsigned* __restrict__ peak, long long ld, int R, int K) {
    const int lane = threadIdx.x & 63, Kp = (K + 31) / 32 * 32;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    const float* p = x + r * ld;
    unsigned m = 0;
    for (int k = 4 * lane; k < K; k += 256) {
        const mh_f4 v = mm_get4<MM_F32>(p + k, K - k);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = hv_max(m, hv_peak(v[j]));
    }
#pragma unroll
    for (int d = 1; d < MH_WAVE; d <<= 1) m = hv_max(m, (unsigned)__shfl_xor((int)m, d, MH_WAVE));
    if (lane == 0) peak[r] = m;
    const int s = hv_shift(m);
    unsigned short* q = y + r * 2 * Kp;
    for (int k = 4 * lane; k < Kp; k += 256) {
        const mh_f4 v = k < K ? mm_get4<MM_F32>(p + k, K - k) : mh_f4{0.f, 0.f, 0.f, 0.f};
        unsigned short* o = q + k / 32 * 64 + k % 32;
        hv_split4(v, make_int4(s, s, s, s), o, o + 32);
    }
}

// Rows [0, R) in groups, cut into pieces of L: by offsets (mm_slot), or (off NULL) E groups of G rows each.
__device__ __forceinline__ bool hv_slot(const int* off, int E, int R, int G, int L, int s, int& e, int& r0, int& r1) {
    if (off) return mm_slot(off, E, R, L, s, e, r0, r1);
    const int per = (G + L - 1) / L;
    e = s / per;
    r0 = e * G + s % per * L;
    r1 = min(r0 + L, (e + 1) * G);
    return e < E;
}

// Columns, first pass: the peaks [E, C] and marks [E, C] (both zero before) of each group's columns, a workgroup for a piece
// of rows and 256 columns.  The largest of integers does not depend on the order of the atomics.  Bound, with the second pass, by
// their bytes: 12 a value, 1,024 x 1,024 weights 5.2 and 5.6 us.
extern "C" __global__ __launch_bounds__(256) void hv_peaks(const float* __restrict__ x, unsigned* __restrict__ peak,
                                                           unsigned* __restrict__ mark, const int* __restrict__ off,
                                                           long long ld, int R, int C, int E, int G, int L) {
    __shared__ unsigned best[4][64][4];
    int e, r0, r1;
    if (!hv_slot(off, E, R, G, L, blockIdx.x, e, r0, r1)) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.y * 256 + 4 * lane;
    unsigned m[4] = {0u, 0u, 0u, 0u};
    if (c < C) {
#pragma unroll 4
        for (int r = r0 + w; r < r1; r += 4) {
            const mh_f4 v = mm_get4<MM_F32>(x + (long long)r * ld + c, C - c);
#pragma unroll
            for (int j = 0; j < 4; ++j) m[j] = hv_max(m[j], hv_peak(v[j]));
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) best[w][lane][j] = m[j];
    __syncthreads();
    const int i = blockIdx.y * 256 + threadIdx.x;        // a column a thread from here on
    if (i >= C) return;
    unsigned b = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) b = hv_max(b, best[k][threadIdx.x >> 2][threadIdx.x & 3]);
    atomicMax(&peak[(long long)e * C + i], b & 0x7FFFFFFFu);
    if (b & HV_ODD) atomicOr(&mark[(long long)e * C + i], HV_ODD);
}

// Columns, second pass: the halves.
extern "C" __global__ __launch_bounds__(256) void hv_columns(const float* __restrict__ x, unsigned short* __restrict__ y,
                                                             const unsigned* __restrict__ peak, const int* __restrict__ off,
                                                             long long ld, int R, int C, int E, int G, int L) {
    int e, r0, r1;
    if (!hv_slot(off, E, R, G, L, blockIdx.x, e, r0, r1)) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.y * 256 + 4 * lane, Cp = (C + 7) / 8 * 8;
    if (c >= Cp) return;
    int4 s = make_int4(0, 0, 0, 0);
    const unsigned* p = peak + (long long)e * C;
    if (c < C) s.x = hv_shift(p[c]);
    if (c + 1 < C) s.y = hv_shift(p[c + 1]);
    if (c + 2 < C) s.z = hv_shift(p[c + 2]);
    if (c + 3 < C) s.w = hv_shift(p[c + 3]);
#pragma unroll 4
    for (int r = r0 + w; r < r1; r += 4) {
        const mh_f4 v = c < C ? mm_get4<MM_F32>(x + (long long)r * ld + c, C - c) : mh_f4{0.f, 0.f, 0.f, 0.f};
        unsigned short* o = y + (long long)r * 2 * Cp + c;
        hv_split4(v, s, o, o + Cp);
    }
}

// A finished tile whose sums stand for sums times 2^(row's shift + column's): what mm_store_tile takes.  Where the tile has
// marked rows or columns (`odd`), the sums are those of the upper halves alone and an unmarked element is taken from C, where
// its own thread put it before.
template <typename tile_t>
struct hv_result {
    static constexpr int ROWS = tile_t::ROWS, COLS = tile_t::COLS;
    const tile_t& t;
    float* C;                                            // the tile's first element, rows N apart
    long long N;
    int rows, cols;
    bool odd = false;
    unsigned a[ROWS];
    mh_u4 b[COLS];
    __device__ __forceinline__ static int row(int i) { return tile_t::row(i); }
    __device__ __forceinline__ static int column(int j) { return tile_t::column(j); }
    // peaks of the tile's rows and columns; their marks apart (ma, mb) or among them (NULL)
    __device__ __forceinline__ hv_result(const tile_t& tile, float* C, long long N, const unsigned* pa, const unsigned* ma,
                                         int rows, const unsigned* pb, const unsigned* mb, int cols)
        : t(tile), C(C), N(N), rows(rows), cols(cols) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int m = min(row(i), rows - 1);
            a[i] = pa[m] | (ma ? ma[m] : 0u);
        }
#pragma unroll
        for (int j = 0; j < COLS; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int n = min(column(j) + c, cols - 1);
                b[j][c] = pb[n] | (mb ? mb[n] : 0u);
            }
    }
    // the whole workgroup's answer; also the barrier after the tile's products
    __device__ __forceinline__ bool any_odd() const {
        unsigned o = 0;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) o |= a[i];
#pragma unroll
        for (int j = 0; j < COLS; ++j) o |= b[j].x | b[j].y | b[j].z | b[j].w;
        return __syncthreads_or((o & HV_ODD) != 0);
    }
    __device__ __forceinline__ mh_f4 scaled(int i, int j) const {
        mh_f4 v = t.value(i, j);
        const int s = hv_shift(a[i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = __builtin_ldexpf(v[c], -(s + hv_shift(b[j][c])));
        return v;
    }
    __device__ __forceinline__ void keep() const {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int j = 0; j < COLS; ++j)
                if (row(i) < rows && column(j) < cols)
                    mm_put4<MM_F32>(C + row(i) * N + column(j), scaled(i, j), cols - column(j));
    }
    __device__ __forceinline__ mh_f4 value(int i, int j) const {
        mh_f4 v = scaled(i, j);
        if (odd) {
            const mh_f4 u = mm_get4<MM_F32>(C + row(i) * N + column(j), cols - column(j));
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = (a[i] | b[j][c]) & HV_ODD ? v[c] : u[c];
        }
        return v;
    }
};

// mm_rows_body on halves: A rows [R][Kp / 32][2][32] with their peaks pa [R]; B either rows, [E][N][Kp / 32][2][32] with pb
// [E][N], or (BS) columns of K contracted rows, [E][K][2][Np] with pb and marks mb [E][N].
// Bound by the matrix cores: 20,000 x 1,024 x 1,024 in 128 us, 980 TFLOP/s of float16 products (three rounds of workgroups where
// 2.45 would do), the cores busy 53 % of it.
template <bool BS, int ACT, typename tile_t>
__device__ __forceinline__ void hv_rows_body(const unsigned short* A, const unsigned short* B, float* C0, const float* bias,
                                             const float* res, float* slope, const int* off, const unsigned* pa,
                                             const unsigned* pb, const unsigned* mb, long long ldr, int R, int N, int K, int E) {
    __shared__ mh_u4 lds[tile_t::LDS];
    const int NT = (N + tile_t::BN - 1) / tile_t::BN, MT = gridDim.x / NT, Kp = (K + 31) / 32 * 32, Np = (N + 7) / 8 * 8;
    int mt, nt, e, r0, r1;
    mm_tile_of(blockIdx.x, gridDim.x, MT, NT, mt, nt);
    const bool live = mm_slot(off, E, R, tile_t::BM, mt, e, r0, r1);
    if (r0 >= R) return;
    const int n0 = nt * tile_t::BN, rows = r1 - r0, cols = min(N - n0, tile_t::BN);
    float* C = C0 + (long long)r0 * N + n0;
    if (!live) {
        for (int i = threadIdx.x; i < rows * cols; i += tile_t::THREADS) C[(long long)(i / cols) * N + i % cols] = 0.f;
        return;
    }
    const unsigned short* a = A + (long long)r0 * 2 * Kp;
    const unsigned short* b = BS ? B + (long long)e * K * 2 * Np + n0 : B + ((long long)e * N + n0) * 2 * Kp;
    const int brows = BS ? min(Np - n0, tile_t::BN) : cols;
    tile_t t;
    t.run(lds, a, 2 * Kp, rows, b, BS ? Np : 2 * Kp, brows, 0, 2 * Kp, BS ? 2 * K : 0);
    const long long col = (long long)e * N + n0;
    hv_result<tile_t> r(t, C, N, pa + r0, nullptr, rows, pb + col, mb ? mb + col : nullptr, cols);
    if (r.any_odd()) {
        r.keep();
        r.odd = true;
        t.template run<true>(lds, a, 2 * Kp, rows, b, BS ? Np : 2 * Kp, brows, 0, 2 * Kp, BS ? 2 * K : 0);
    }
    bias = bias ? bias + (long long)e * N : nullptr;
    if (n0 + tile_t::BN <= N) mm_store_tile<MM_F32, ACT, true>(r, r0, rows, n0, N, bias, res, ldr, slope, C0);
    else mm_store_tile<MM_F32, ACT, false>(r, r0, rows, n0, N, bias, res, ldr, slope, C0);
}

// mm_outer_body on halves: A columns [R][2][Mp], B columns [R][2][Np], peaks and marks [E][M] and [E][N].
template <typename tile_t>
__device__ __forceinline__ void hv_outer_body(const unsigned short* A, const unsigned short* B, float* C0, float* part,
                                              const int* off, const unsigned* pa, const unsigned* ma, const unsigned* pb,
                                              const unsigned* mb, int R, int M, int N, int E, int L) {
    __shared__ mh_u4 lds[tile_t::LDS];
    const int NT = (N + tile_t::BN - 1) / tile_t::BN, MT = gridDim.x / NT, Mp = (M + 7) / 8 * 8, Np = (N + 7) / 8 * 8;
    int mt, nt, e = 0, r0 = 0, r1 = R;
    mm_tile_of(blockIdx.x, gridDim.x, MT, NT, mt, nt);
    if (L) {
        if (!mm_slot(off, E, R, L, blockIdx.y, e, r0, r1)) return;
    } else if (off) {
        e = mm_by_length(off, E, blockIdx.y);
        r0 = min(max(off[e], 0), R);
        r1 = min(max(off[e + 1], r0), R);
    }
    const int m0 = mt * tile_t::BM, n0 = nt * tile_t::BN, rows = min(M - m0, tile_t::BM), cols = min(N - n0, tile_t::BN);
    const unsigned short *a = A + (long long)r0 * 2 * Mp + m0, *b = B + (long long)r0 * 2 * Np + n0;
    const int ar = min(Mp - m0, tile_t::BM), br = min(Np - n0, tile_t::BN);
    tile_t t;
    t.run(lds, a, Mp, ar, b, Np, br, 0, 2 * (r1 - r0));
    float* C = (L ? part + (long long)blockIdx.y * M * N : C0 + (long long)e * M * N) + (long long)m0 * N + n0;
    const long long ra = (long long)e * M + m0, rb = (long long)e * N + n0;
    hv_result<tile_t> r(t, C, N, pa + ra, ma + ra, rows, pb + rb, mb + rb, cols);
    if (r.any_odd()) {
        r.keep();
        r.odd = true;
        t.template run<true>(lds, a, Mp, ar, b, Np, br, 0, 2 * (r1 - r0));
    }
#pragma unroll
    for (int i = 0; i < tile_t::ROWS; ++i)
#pragma unroll
        for (int j = 0; j < tile_t::COLS; ++j)
            if (tile_t::row(i) < rows && tile_t::column(j) < cols)
                mm_put4<MM_F32>(C + (long long)tile_t::row(i) * N + tile_t::column(j), r.value(i, j),
                                cols - tile_t::column(j));
}
