// mh_experts.h — rows to their places in the order by expert and back, prepended with mh_device.h and mh_matmul.h.
//
// place[t k + j]: where assignment j of node t stands among the A = T k places (-1: dropped), as mh_expert_order.h makes it;
// the places behind offsets[E] belong to no assignment.
#pragma once

// A thread group of 2^lg lanes per row; rows past the last group are zeroed by every block in turn.  A row's number and the
// step to the next take 64 bits: A, up to 2^31, and the number of thread groups add up to more than 32 hold.
template <int TY>
__device__ __forceinline__ void ex_zero_tail(typename mm_type<TY>::t* y, const int* offsets, int E, int A, int C, int lg) {
    typedef mm_vec<TY> vec;
    vec z;
    z.zero();
    const int tpr = 1 << lg, l = threadIdx.x & (tpr - 1);
    const long long rpb = blockDim.x >> lg;
    for (long long p = min(max(offsets[E], 0), A) + blockIdx.x * rpb + (threadIdx.x >> lg); p < A; p += gridDim.x * rpb)
        for (int c = l * vec::V; c < C; c += tpr * vec::V) z.put(y + p * C + c, C - c);
}

// y[place[t, j]] = x[t]: each row of x read once, written to its places past the caches (here and below: a training step's
// four passes over 32,768 nodes of four rows of 1,024 bfloat16 values took 350 us with ordinary stores, 276 with these).  Bound
// by its bytes: 63 us there, 5.3 TB/s.
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
                if (p >= 0 && p < A) v.template put<true>(y + (long long)p * C + c, C - c);
            }
        }
    ex_zero_tail<TY>(y, offsets, E, A, C, lg);
}

// out[t] = res[t] + sum over the kept j of w[t, j] y[place[t, j]] (w NULL: 1), j in order.  Bound by its bytes: a node's rows
// lie anywhere, so four are loaded before the first is added, and rows and results pass by the caches: 52 us at 32,768 nodes
// of four rows of 1,024 bfloat16 values, 6.5 TB/s (ordinary accesses: 80).
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
        for (int j0 = 0; j0 < k; j0 += 4) {
            int p[4];
            float q[4];
            mh_u4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = t * k + min(j0 + j, k - 1);
                p[j] = j0 + j < k ? place[at] : -1;
                q[j] = w ? w[at] : 1.f;
                if (p[j] >= A) p[j] = -1;
            }
            // without a branch: a dropped one loads row 0 and is not added, whatever that holds
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = vec::template raw<true>(static_cast<const S*>(y_) + (long long)max(p[j], 0) * C + c, C - c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                vec x;
                x.set(v[j]);
#pragma unroll
                for (int i = 0; i < vec::V; ++i) s.v[i] = p[j] >= 0 ? __builtin_fmaf(q[j], x.v[i], s.v[i]) : s.v[i];
            }
        }
        s.template put<true>(static_cast<S*>(out_) + t * C + c, C - c);
    }
}

// dy[place[t, j]] = w[t, j] g[t] (dy NULL: not wanted) and dw[t, j] = <g[t], y[place[t, j]]>, 0 where dropped (dw NULL: not
// wanted), four j at a time: a vector of g is loaded once for the four rows of y and dy, which pass by the caches.  Bound by its
// bytes: 114 us at 32,768 nodes of four rows of 1,024 bfloat16 values, 5.3 TB/s.
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
        for (int j0 = 0; j0 < k; j0 += 4) {
            int p[4];
            float q[4], s[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = t * k + min(j0 + j, k - 1);
                p[j] = j0 + j < k ? place[at] : -1;
                q[j] = w ? w[at] : 1.f;
                s[j] = 0.f;
                if (p[j] >= A) p[j] = -1;
            }
            for (int c = l * vec::V; c < C; c += tpr * vec::V) {
                const mh_u4 gr = vec::raw(static_cast<const S*>(g_) + t * ldg + c, C - c);
                mh_u4 yr[4];
                if (dw)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        yr[j] = vec::template raw<true>(static_cast<const S*>(y_) + (long long)max(p[j], 0) * C + c, C - c);
                vec g;
                g.set(gr);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (p[j] < 0) continue;
                    if (dw) {
                        vec y;
                        y.set(yr[j]);
#pragma unroll
                        for (int i = 0; i < vec::V; ++i) s[j] += g.v[i] * y.v[i];
                    }
                    if (dy_) {
                        vec d;
#pragma unroll
                        for (int i = 0; i < vec::V; ++i) d.v[i] = g.v[i] * q[j];
                        d.template put<true>(static_cast<S*>(dy_) + (long long)p[j] * C + c, C - c);
                    }
                }
            }
            if (dw)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    for (int d = tpr >> 1; d; d >>= 1) s[j] += __shfl_xor(s[j], d, MH_WAVE);
                    if (l == 0 && j0 + j < k) dw[t * k + j0 + j] = s[j];
                }
        }
    if (dy_) ex_zero_tail<TY>(static_cast<S*>(dy_), offsets, E, A, C, lg);
}
