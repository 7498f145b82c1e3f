// mh_experts.h — rows to their places in the order by expert and back, prepended with mh_device.h and mh_matmul.h.
//
// place[t k + j]: where assignment j of node t stands among the A = T k places (-1: dropped), as mh_expert_order.h makes it;
// the places behind offsets[E] belong to no assignment.
#pragma once

// A thread group of 2^lg lanes per row; rows past the last group are zeroed by every block in turn.
template <int TY>
__device__ __forceinline__ void ex_zero_tail(typename mm_type<TY>::t* y, const int* offsets, int E, int A, int C, int lg) {
    typedef mm_vec<TY> vec;
    vec z;
    z.zero();
    const int tpr = 1 << lg, l = threadIdx.x & (tpr - 1), rpb = blockDim.x >> lg;
    for (int p = min(max(offsets[E], 0), A) + (int)blockIdx.x * rpb + (threadIdx.x >> lg); p < A; p += gridDim.x * rpb)
        for (int c = l * vec::V; c < C; c += tpr * vec::V) z.put(y + (long long)p * C + c, C - c);
}

// y[place[t, j]] = x[t]: each row of x read once, written to its places
template <int TY>
__device__ __forceinline__ void ex_dispatch_body(const void* x_, const int* place, const int* offsets, void* y_, long long ldx,
                                                 int T, int k, int C, int E, int lg) {
    typedef mm_vec<TY> vec;
    typedef typename mm_type<TY>::t S;
    S* y = static_cast<S*>(y_);
    const int tpr = 1 << lg, l = threadIdx.x & (tpr - 1);
    const long long t = (long long)blockIdx.x * (blockDim.x >> lg) + (threadIdx.x >> lg);
    const int A = T * k;
    if (t < T)
        for (int c = l * vec::V; c < C; c += tpr * vec::V) {
            vec v;
            v.get(static_cast<const S*>(x_) + t * ldx + c, C - c);
            for (int j = 0; j < k; ++j) {
                const int p = place[t * k + j];
                if (p >= 0 && p < A) v.put(y + (long long)p * C + c, C - c);
            }
        }
    ex_zero_tail<TY>(y, offsets, E, A, C, lg);
}

// out[t] = res[t] + sum over the kept j of w[t, j] y[place[t, j]] (w NULL: 1), j in order
template <int TY>
__device__ __forceinline__ void ex_combine_body(const void* y_, const float* w, const int* place, const void* res_, void* out_,
                                                long long ldr, int T, int k, int C, int lg) {
    typedef mm_vec<TY> vec;
    typedef typename mm_type<TY>::t S;
    const int tpr = 1 << lg, l = threadIdx.x & (tpr - 1);
    const long long t = (long long)blockIdx.x * (blockDim.x >> lg) + (threadIdx.x >> lg);
    const int A = T * k;
    if (t >= T) return;
    for (int c = l * vec::V; c < C; c += tpr * vec::V) {
        vec s;
        if (res_) s.get(static_cast<const S*>(res_) + t * ldr + c, C - c);
        else s.zero();
        for (int j = 0; j < k; ++j) {
            const int p = place[t * k + j];
            if (p < 0 || p >= A) continue;
            vec v;
            v.get(static_cast<const S*>(y_) + (long long)p * C + c, C - c);
            const float q = w ? w[t * k + j] : 1.f;
#pragma unroll
            for (int i = 0; i < vec::V; ++i) s.v[i] += q * v.v[i];
        }
        s.put(static_cast<S*>(out_) + t * C + c, C - c);
    }
}

// dy[place[t, j]] = w[t, j] g[t] (dy NULL: not wanted) and dw[t, j] = <g[t], y[place[t, j]]>, 0 where dropped (dw NULL: not
// wanted); each row of g is read once per j from the caches
template <int TY>
__device__ __forceinline__ void ex_combine_bwd_body(const void* g_, const void* y_, const float* w, const int* place,
                                                    const int* offsets, void* dy_, float* dw, long long ldg, int T, int k, int C,
                                                    int E, int lg) {
    typedef mm_vec<TY> vec;
    typedef typename mm_type<TY>::t S;
    const int tpr = 1 << lg, l = threadIdx.x & (tpr - 1);
    const long long t = (long long)blockIdx.x * (blockDim.x >> lg) + (threadIdx.x >> lg);
    const int A = T * k;
    if (t < T)
        for (int j = 0; j < k; ++j) {
            const int p = place[t * k + j];
            const bool kept = p >= 0 && p < A;
            const float q = w ? w[t * k + j] : 1.f;
            float s = 0.f;
            if (kept)
                for (int c = l * vec::V; c < C; c += tpr * vec::V) {
                    vec g;
                    g.get(static_cast<const S*>(g_) + t * ldg + c, C - c);
                    if (dw) {
                        vec y;
                        y.get(static_cast<const S*>(y_) + (long long)p * C + c, C - c);
#pragma unroll
                        for (int i = 0; i < vec::V; ++i) s += g.v[i] * y.v[i];
                    }
                    if (dy_) {
#pragma unroll
                        for (int i = 0; i < vec::V; ++i) g.v[i] *= q;
                        g.put(static_cast<S*>(dy_) + (long long)p * C + c, C - c);
                    }
                }
            if (dw) {
                for (int d = tpr >> 1; d; d >>= 1) s += __shfl_xor(s, d, MH_WAVE);
                if (l == 0) dw[t * k + j] = s;
            }
        }
    if (dy_) ex_zero_tail<TY>(static_cast<S*>(dy_), offsets, E, A, C, lg);
}
