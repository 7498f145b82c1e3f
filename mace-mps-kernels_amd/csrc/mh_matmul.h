// mh_matmul.h — matrix products of the trainable node layers (dense, expert_dense), prepended with mh_device.h.
//
// One body computes D[m, n] = sum_k A[m, k] B[n, k] on the matrix cores for the three products of a layer
// y = act(x W^T + b) + r, x [T, K], W [N, K]:
//   forward   D = y,   A = x            B = W             both contiguous along the contraction k
//   input     D = dx,  A = p [T, N]     B = W^T           A contiguous along it, B strided
//   weights   D = dW,  A = p^T          B = x^T           both strided (the contraction runs over rows)
// with p = dL/dy act'(a).  bf16 and fp16 operands feed v_mfma_f32_16x16x32 as they are; a float32 operand is split into
// three bf16 parts as a tile enters LDS (mh_split8), and of the nine products of parts the six leading ones are kept:
// the terms left out are below 2^-24 of |a b|.  hi*hi has an accumulator of its own: an infinite or NaN operand makes it
// exactly what a float32 sum would be, while the lower parts of such an operand (inf - inf) are meaningless, so the
// store takes the sum of both accumulators only where the first is finite.  Sums are float32 throughout.
#pragma once

#define MM_F32 0
#define MM_BF16 1
#define MM_F16 2

typedef _Float16 mh_h8 __attribute__((ext_vector_type(8)));

// Unaligned 4-, 8- and 16-byte accesses: one instruction each on gfx950 whatever the address, so rows of odd lengths
// need no path of their own.
typedef unsigned mh_u1x __attribute__((aligned(2)));
typedef unsigned mh_u2x __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned mh_u4x __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned mh_u2 __attribute__((ext_vector_type(2)));

template <int TY> struct mm_type { typedef unsigned short t; };
template <> struct mm_type<MM_F32> { typedef float t; };

template <int TY>
__device__ __forceinline__ float mm_get(const typename mm_type<TY>::t* p) {
    if constexpr (TY == MM_F32) return *p;
    else if constexpr (TY == MM_BF16) return __uint_as_float((unsigned)*p << 16);
    else return (float)__builtin_bit_cast(_Float16, *p);
}

template <int TY>
__device__ __forceinline__ float mm_widen(unsigned short v) {
    if constexpr (TY == MM_BF16) return __uint_as_float((unsigned)v << 16);
    else return (float)__builtin_bit_cast(_Float16, v);
}

// rounds to nearest even
template <int TY>
__device__ __forceinline__ unsigned short mm_round(float v) {
    if constexpr (TY == MM_BF16) return __builtin_bit_cast(unsigned short, (__bf16)v);
    else return __builtin_bit_cast(unsigned short, (_Float16)v);
}

// four consecutive elements as floats, and back
template <int TY>
__device__ __forceinline__ mh_f4 mm_get4(const typename mm_type<TY>::t* p) {
    if constexpr (TY == MM_F32) {
        return __builtin_bit_cast(mh_f4, (mh_u4) * reinterpret_cast<const mh_u4x*>(p));
    } else {
        const mh_u2 v = *reinterpret_cast<const mh_u2x*>(p);
        return mh_f4{mm_widen<TY>((unsigned short)v.x), mm_widen<TY>((unsigned short)(v.x >> 16)),
                     mm_widen<TY>((unsigned short)v.y), mm_widen<TY>((unsigned short)(v.y >> 16))};
    }
}

template <int TY>
__device__ __forceinline__ void mm_put4(typename mm_type<TY>::t* p, mh_f4 v) {
    if constexpr (TY == MM_F32) {
        *reinterpret_cast<mh_u4x*>(p) = __builtin_bit_cast(mh_u4, v);
    } else {
        *reinterpret_cast<mh_u2x*>(p) = mh_u2{mm_round<TY>(v.x) | (unsigned)mm_round<TY>(v.y) << 16,
                                              mm_round<TY>(v.z) | (unsigned)mm_round<TY>(v.w) << 16};
    }
}

// `n` elements (1 to 4) at p; the others are zero / left alone
template <int TY>
__device__ __forceinline__ mh_f4 mm_get4(const typename mm_type<TY>::t* p, int n) {
    if (n >= 4) return mm_get4<TY>(p);
    mh_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < n) v[j] = mm_get<TY>(p + j);
    return v;
}

template <int TY>
__device__ __forceinline__ void mm_put4(typename mm_type<TY>::t* p, mh_f4 v, int n) {
    if (n >= 4) return mm_put4<TY>(p, v);
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < n) {
            if constexpr (TY == MM_F32) p[j] = v[j];
            else p[j] = mm_round<TY>(v[j]);
        }
}

// Sixteen bytes of a row at a time: V elements, as floats.  `n`: elements that the row has from p on.
template <int TY>
struct mm_vec {
    static constexpr int V = TY == MM_F32 ? 4 : 8;
    float v[V];
    __device__ __forceinline__ void get(const typename mm_type<TY>::t* p, int n) {
        if (n >= V) {
            const mh_u4 w = *reinterpret_cast<const mh_u4x*>(p);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (TY == MM_F32) v[j] = __uint_as_float(w[j]);
                else v[j] = mm_widen<TY>((unsigned short)(w[j / 2] >> (16 * (j & 1))));
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = j < n ? mm_get<TY>(p + j) : 0.f;
        }
    }
    __device__ __forceinline__ void put(typename mm_type<TY>::t* p, int n) const {
        if (n >= V) {
            mh_u4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (TY == MM_F32) w[j] = __float_as_uint(v[j]);
                else w[j] = mm_round<TY>(v[2 * j]) | (unsigned)mm_round<TY>(v[2 * j + 1]) << 16;
            }
            *reinterpret_cast<mh_u4x*>(p) = w;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) {
                    if constexpr (TY == MM_F32) p[j] = v[j];
                    else p[j] = mm_round<TY>(v[j]);
                }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = 0.f;
    }
};

// ------------------------------------------------------------------------------------------------ activations
#define MM_NONE 0
#define MM_RELU 1
#define MM_SILU 2
#define MM_GELU 3

// relu keeps NaN (comparisons with it are false); silu(a) = a / (1 + e^-a); gelu(a) = a Phi(a), Phi the normal
// distribution function by erf
__device__ __forceinline__ float mm_act(int act, float a) {
    if (act == MM_RELU) return a < 0.f ? 0.f : a;
    if (act == MM_SILU) return a / (1.f + expf(-a));
    if (act == MM_GELU) return 0.5f * a * (1.f + erff(a * 0.70710678f));
    return a;
}

__device__ __forceinline__ float mm_act_slope(int act, float a) {
    if (act == MM_RELU) return a > 0.f ? 1.f : 0.f;
    if (act == MM_SILU) {
        const float q = 1.f / (1.f + expf(-a));
        return q * (1.f + a * (1.f - q));
    }
    if (act == MM_GELU) return 0.5f * (1.f + erff(a * 0.70710678f)) + a * 0.39894228f * expf(-0.5f * a * a);
    return 1.f;
}

// act'(a) as the forward keeps it for the backward: float32, or for the 16-bit types fixed point with steps of 2^-15 from
// -0.5 (the slopes of all activations lie in [-0.13, 1.13]; 0 and 1 are exact; 65535 stands for NaN): its error of 2^-16
// is far below the 2^-8 (2^-11) to which these types round the product p, where a slope kept in them would add its own.
__device__ __forceinline__ unsigned mm_slope_code(float d) {
    return d == d ? (unsigned)__float2int_rn((d + 0.5f) * 32768.f) : 65535u;
}
__device__ __forceinline__ float mm_slope_value(unsigned c) {
    return c == 65535u ? __uint_as_float(0x7FC00000u) : (float)(int)c * 3.0517578125e-5f - 0.5f;
}

// ------------------------------------------------------------------------------------------------ groups of rows
// Rows [0, R) in E groups, group e from off[e] to off[e + 1]; each group is cut into pieces of L rows, and slot s is the
// s-th piece.  False past the last one; rows after the last group then follow as pieces with e = -1.  off NULL: one group
// of all rows.  Offsets are clamped into [0, R] and to the largest before them, so whatever they hold, groups are disjoint,
// no piece leads out of the tensors, and there are at most R / L + E of them.  Every lane of a wave calls (64 groups at a
// time are scanned across it); R + L < 2^31.
__device__ __forceinline__ bool mm_slot(const int* __restrict__ off, int E, int R, int L, int s, int& e, int& r0, int& r1) {
    if (!off) {
        e = 0;
        r0 = s * L;
        r1 = min(R, r0 + L);
        return r0 < R;
    }
    const int lane = threadIdx.x & (MH_WAVE - 1);
    int base = 0, top = min(max(off[0], 0), R);          // pieces and rows before these 64 groups
    for (int g0 = 0; g0 < E; g0 += MH_WAVE) {
        int hi = max(top, min(off[min(g0 + lane, E - 1) + 1], R));
#pragma unroll
        for (int d = 1; d < MH_WAVE; d <<= 1) {
            const int t = __shfl_up(hi, d, MH_WAVE);
            if (lane >= d) hi = max(hi, t);
        }
        const int prev = __shfl_up(hi, 1, MH_WAVE), lo = lane ? prev : top;
        const int n = g0 + lane < E ? (hi - lo + L - 1) / L : 0;
        int inc = n;
#pragma unroll
        for (int d = 1; d < MH_WAVE; d <<= 1) {
            const int t = __shfl_up(inc, d, MH_WAVE);
            if (lane >= d) inc += t;
        }
        const int total = mh_bcast(inc, MH_WAVE - 1);
        if (s < base + total) {
            const int l = __ffsll((unsigned long long)__ballot(base + inc > s)) - 1;
            const int glo = mh_bcast(lo, l), ghi = mh_bcast(hi, l), before = mh_bcast(inc - n, l);
            e = g0 + l;
            r0 = glo + (s - base - before) * L;
            r1 = min(ghi, r0 + L);
            return true;
        }
        base += total;
        top = mh_bcast(hi, MH_WAVE - 1);
    }
    e = -1;
    const long long r = top + (long long)(s - base) * L;
    r0 = (int)min(r, (long long)R);
    r1 = min(R, r0 + L);
    return false;
}

// ------------------------------------------------------------------------------------------------ operand tiles
// A tile of ROWS x BK values of an operand in LDS: octets of eight values along k, 16 bytes each (one plane for the 16-bit
// types, three for the parts of float32), octet o of row r at r OPR + (o ^ swizzle(r)).  The swizzle gives 16 rows that
// are read at one o sixteen different places of LDS's 256 bytes of banks.
template <int OPR>
__device__ __forceinline__ int mm_place(int row, int o) {
    return row * OPR + (o ^ ((row / (16 / OPR)) & (OPR - 1)));
}

// One operand as its threads load it: STRIDED false, element (row, k) at p[row ld + k]; true, at p[k ld + row].  Rows past
// `rows` repeat the last one (their results are never stored); k past `kend` gives zeros in both operands.
template <int TY, bool STRIDED, int ROWS, int BK, int THREADS>
struct mm_loader {
    typedef typename mm_type<TY>::t T;
    static constexpr int OPR = BK / 8;
    static constexpr int PAIR = (STRIDED && TY != MM_F32) ? 2 : 1;       // rows a thread loads together
    static constexpr int ITEMS = ROWS * OPR / PAIR / THREADS;
    static constexpr int WORDS = TY == MM_F32 ? 8 : 4 * PAIR;            // 32-bit words of an item
    static constexpr int PLANES = TY == MM_F32 ? 3 : 1;
    static_assert(ROWS * OPR / PAIR % THREADS == 0, "a tile is a whole number of items per thread");
    unsigned w[ITEMS][STRIDED && TY != MM_F32 ? 8 : WORDS];
    const T* p;
    long long ld;
    int rows;

    __device__ __forceinline__ void init(const T* base, long long stride, int nrows) {
        p = base;
        ld = stride;
        rows = nrows;
    }
    __device__ __forceinline__ static void where(int j, int& row, int& o) {
        const int i = threadIdx.x + j * THREADS;
        if constexpr (STRIDED) {
            row = i % (ROWS / PAIR) * PAIR;
            o = i / (ROWS / PAIR);
        } else {
            row = i / OPR;
            o = i % OPR;
        }
    }
    __device__ __forceinline__ void load(int k0, int kend) {
        const bool whole = k0 + BK <= kend;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            int row, o;
            where(j, row, o);
            const int k = k0 + 8 * o;
            if constexpr (!STRIDED) {
                const T* q = p + (long long)min(row, rows - 1) * ld + k;
                if (whole || k + 8 <= kend) {
#pragma unroll
                    for (int h = 0; h < WORDS / 4; ++h) {
                        const mh_u4 v = reinterpret_cast<const mh_u4x*>(q)[h];
#pragma unroll
                        for (int c = 0; c < 4; ++c) w[j][4 * h + c] = v[c];
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < WORDS; ++c) {
                        if constexpr (TY == MM_F32) {
                            w[j][c] = k + c < kend ? __float_as_uint(q[c]) : 0u;
                        } else {
                            const unsigned lo = k + 2 * c < kend ? q[2 * c] : 0u;
                            const unsigned hi = k + 2 * c + 1 < kend ? q[2 * c + 1] : 0u;
                            w[j][c] = lo | hi << 16;
                        }
                    }
                }
            } else {
                // the pair past an odd count's end: its two rows one by one
                const bool both = PAIR == 1 || row + 1 < rows;
                const T* q = p + min(row, rows - 1);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const bool in = whole || k + c < kend;
                    const T* qc = q + (long long)(in ? k + c : 0) * ld;
                    unsigned v = 0;
                    if (in) {
                        if constexpr (TY == MM_F32) v = __float_as_uint(*qc);
                        else v = both ? (unsigned)*reinterpret_cast<const mh_u1x*>(qc) : (unsigned)*qc;
                    }
                    w[j][c] = v;
                }
            }
        }
    }
    // the loaded items into an LDS tile of PLANES planes of `plane` octets each
    __device__ __forceinline__ void store(mh_u4* tile) const {
        constexpr int plane = ROWS * OPR;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            int row, o;
            where(j, row, o);
            if constexpr (TY == MM_F32) {
                float v[8];
                mh_bf8 s[3];
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = __uint_as_float(w[j][c]);
                mh_split8(v, s);
#pragma unroll
                for (int q = 0; q < 3; ++q) tile[q * plane + mm_place<OPR>(row, o)] = __builtin_bit_cast(mh_u4, s[q]);
            } else if constexpr (!STRIDED) {
                tile[mm_place<OPR>(row, o)] = mh_u4{w[j][0], w[j][1], w[j][2], w[j][3]};
            } else {
                mh_u4 a, b;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    a[c] = (w[j][2 * c] & 0xFFFFu) | w[j][2 * c + 1] << 16;
                    b[c] = w[j][2 * c] >> 16 | (w[j][2 * c + 1] & 0xFFFF0000u);
                }
                tile[mm_place<OPR>(row, o)] = a;
                tile[mm_place<OPR>(row + 1, o)] = b;
            }
        }
    }
};

template <int TY>
__device__ __forceinline__ mh_f4 mm_mfma(mh_u4 a, mh_u4 b, mh_f4 c) {
    if constexpr (TY == MM_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mh_h8, a), __builtin_bit_cast(mh_h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mh_bf8, a), __builtin_bit_cast(mh_bf8, b), c, 0, 0,
                                                       0);
}

// The sums of one workgroup's tile over k in [kbeg, kend): WM x WN waves, each FM x FN fragments of 16 x 16.  B's fragment
// is the instruction's first operand, so that a lane ends with four consecutive n (4 (lane / 16) + j) of one m
// (lane % 16) and stores them at once.  BUFS LDS buffers; the loads of the next tile are in flight during a tile's
// products.
template <int TY, bool AS, bool BS, int WM, int WN, int FM, int FN, int BK, int BUFS>
struct mm_tile {
    typedef typename mm_type<TY>::t T;
    static constexpr int THREADS = 64 * WM * WN, BM = 16 * FM * WM, BN = 16 * FN * WN, OPR = BK / 8;
    static constexpr int PLANES = TY == MM_F32 ? 3 : 1;
    static constexpr int TA = PLANES * BM * OPR, TB = PLANES * BN * OPR;      // octets of a buffer
    static constexpr int LDS = BUFS * (TA + TB);
    mh_f4 acc[FM][FN];
    mh_f4 low[TY == MM_F32 ? FM : 1][TY == MM_F32 ? FN : 1];                 // the products below hi hi

    __device__ __forceinline__ void products(const mh_u4* a, const mh_u4* b) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int ra = (wave / WN) * 16 * FM + (lane & 15), rb = (wave % WN) * 16 * FN + (lane & 15), q = lane >> 4;
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) {
            mh_u4 fa[FM][PLANES], fb[FN][PLANES];
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int s = 0; s < PLANES; ++s) fa[i][s] = a[s * BM * OPR + mm_place<OPR>(ra + 16 * i, 4 * ks + q)];
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int s = 0; s < PLANES; ++s) fb[i][s] = b[s * BN * OPR + mm_place<OPR>(rb + 16 * i, 4 * ks + q)];
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    acc[i][j] = mm_mfma<TY>(fb[j][0], fa[i][0], acc[i][j]);
                    if constexpr (TY == MM_F32) {
                        low[i][j] = mm_mfma<TY>(fb[j][0], fa[i][2], low[i][j]);
                        low[i][j] = mm_mfma<TY>(fb[j][1], fa[i][1], low[i][j]);
                        low[i][j] = mm_mfma<TY>(fb[j][2], fa[i][0], low[i][j]);
                        low[i][j] = mm_mfma<TY>(fb[j][0], fa[i][1], low[i][j]);
                        low[i][j] = mm_mfma<TY>(fb[j][1], fa[i][0], low[i][j]);
                    }
                }
        }
    }

    __device__ __forceinline__ void run(mh_u4* lds, const T* A, long long lda, int arows, const T* B, long long ldb, int brows,
                                        int kbeg, int kend) {
        mm_loader<TY, AS, BM, BK, THREADS> la;
        mm_loader<TY, BS, BN, BK, THREADS> lb;
        la.init(A, lda, arows);
        lb.init(B, ldb, brows);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                acc[i][j] = mh_f4{0.f, 0.f, 0.f, 0.f};
                if constexpr (TY == MM_F32) low[i][j] = mh_f4{0.f, 0.f, 0.f, 0.f};
            }
        if (kbeg >= kend) return;                       // uniform over the workgroup
        la.load(kbeg, kend);
        lb.load(kbeg, kend);
        la.store(lds);
        lb.store(lds + BUFS * TA);
        __syncthreads();
        int cur = 0;
        for (int k = kbeg; k < kend; k += BK) {
            const bool more = k + BK < kend;
            if (more) {
                la.load(k + BK, kend);
                lb.load(k + BK, kend);
            }
            products(lds + cur * TA, lds + BUFS * TA + cur * TB);
            if (!more) break;
            if (BUFS == 1) __syncthreads();             // one buffer: every wave has read it
            else cur ^= 1;
            la.store(lds + cur * TA);
            lb.store(lds + BUFS * TA + cur * TB);
            __syncthreads();
        }
    }

    // Calls f(m, n, sums of D[m, n .. n + 3]) for the lane's fragments, m and n within the tile.
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int m0 = (wave / WN) * 16 * FM + (lane & 15), n0 = (wave % WN) * 16 * FN + 4 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                mh_f4 v = acc[i][j];
                if constexpr (TY == MM_F32) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        v[c] = __builtin_isfinite(v[c]) ? v[c] + low[i][j][c] : v[c];
                }
                f(m0 + 16 * i, n0 + 16 * j, v);
            }
    }
};

// The tile (mt, nt) of a block among MT x NT: bands of eight row tiles, walked column by column, in one contiguous range
// per XCD, so that blocks which share an L2 share operand tiles.
__device__ __forceinline__ void mm_tile_of(int b, int blocks, int MT, int NT, int& mt, int& nt) {
    const int l = mh_xcd_block(b, blocks), band = 8 * NT, first = l / band * 8, high = min(8, MT - first), i = l % band;
    mt = first + i % high;
    nt = i / high;
}

// Forward and input gradient: R rows of A [R, K] in groups, B the group's weights ([N, K], or [K, N] where BS), the
// epilogue v = sums + bias[e]; slope = act'(v); C = act(v) + res.  Rows of no group are written as zeros.
template <int TY, bool BS, int WM, int WN, int FM, int FN, int BK, int BUFS>
__device__ __forceinline__ void mm_rows_body(const void* A_, const void* B_, void* C_, const void* bias_, const void* res_,
                                             void* slope_, const int* off, long long lda, long long ldr, int R, int N, int K,
                                             int E, int act) {
    typedef mm_tile<TY, false, BS, WM, WN, FM, FN, BK, BUFS> tile_t;
    typedef typename mm_type<TY>::t T;
    __shared__ mh_u4 lds[tile_t::LDS];
    const int NT = (N + tile_t::BN - 1) / tile_t::BN, MT = gridDim.x / NT;
    int mt, nt, e, r0, r1;
    mm_tile_of(blockIdx.x, gridDim.x, MT, NT, mt, nt);
    const bool live = mm_slot(off, E, R, tile_t::BM, mt, e, r0, r1);
    if (r0 >= R) return;
    const int n0 = nt * tile_t::BN, rows = r1 - r0;
    T* C = static_cast<T*>(C_) + (long long)r0 * N + n0;
    tile_t t;
    if (!live) {
        // a tail of rows without a group
        for (int i = threadIdx.x; i < rows * min(N - n0, tile_t::BN); i += tile_t::THREADS) {
            const int w = min(N - n0, tile_t::BN);
            C[(long long)(i / w) * N + i % w] = 0;
        }
        return;
    }
    const T* A = static_cast<const T*>(A_) + (long long)r0 * lda;
    const T* B = static_cast<const T*>(B_) + (long long)e * N * K + (BS ? (long long)n0 : (long long)n0 * K);
    t.run(lds, A, lda, rows, B, BS ? N : K, min(N - n0, tile_t::BN), 0, K);
    const T* bias = bias_ ? static_cast<const T*>(bias_) + (long long)e * N + n0 : nullptr;
    const T* res = res_ ? static_cast<const T*>(res_) + (long long)r0 * ldr + n0 : nullptr;
    t.each([&](int m, int n, mh_f4 v) {
        const int c = N - n0 - n;                       // columns that exist from here on
        if (m >= rows || c <= 0) return;
        if (bias) v += mm_get4<TY>(bias + n, c);
        if (slope_) {
            const long long at = ((long long)r0 + m) * N + n0 + n;
            mh_f4 d;
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = mm_act_slope(act, v[j]);
            if constexpr (TY == MM_F32) {
                mm_put4<MM_F32>(static_cast<float*>(slope_) + at, d, c);
            } else {
                unsigned short* s = static_cast<unsigned short*>(slope_) + at;
                if (c >= 4)
                    *reinterpret_cast<mh_u2x*>(s) = mh_u2{mm_slope_code(d[0]) | mm_slope_code(d[1]) << 16,
                                                          mm_slope_code(d[2]) | mm_slope_code(d[3]) << 16};
                else
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        if (j < c) s[j] = (unsigned short)mm_slope_code(d[j]);
            }
        }
        if (act != MM_NONE)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = mm_act(act, v[j]);
        if (res) v += mm_get4<TY>(res + (long long)m * ldr + n, c);
        mm_put4<TY>(C + (long long)m * N + n, v, c);
    });
}

// Weight gradients: D[e] [M, N] = sum over the group's rows of A[r, m] B[r, n] (A = p [R, M], B = x [R, N]).  blockIdx.y is
// the group (L 0: all its rows; none give zeros), or a slot of at most L of its rows whose sums go to part[slot] in float32.
template <int TY, int WM, int WN, int FM, int FN, int BK, int BUFS>
__device__ __forceinline__ void mm_outer_body(const void* A_, const void* B_, void* C_, float* part, const int* off,
                                              long long lda, long long ldb, int R, int M, int N, int E, int L) {
    typedef mm_tile<TY, true, true, WM, WN, FM, FN, BK, BUFS> tile_t;
    typedef typename mm_type<TY>::t T;
    __shared__ mh_u4 lds[tile_t::LDS];
    const int NT = (N + tile_t::BN - 1) / tile_t::BN, MT = gridDim.x / NT;
    int mt, nt, e = 0, r0 = 0, r1 = R;
    mm_tile_of(blockIdx.x, gridDim.x, MT, NT, mt, nt);
    if (L) {
        if (!mm_slot(off, E, R, L, blockIdx.y, e, r0, r1)) return;
    } else if (off) {
        e = blockIdx.y;
        r0 = min(max(off[e], 0), R);
        r1 = min(max(off[e + 1], r0), R);
    }
    const int m0 = mt * tile_t::BM, n0 = nt * tile_t::BN;
    tile_t t;
    t.run(lds, static_cast<const T*>(A_) + (long long)r0 * lda + m0, lda, min(M - m0, tile_t::BM),
          static_cast<const T*>(B_) + (long long)r0 * ldb + n0, ldb, min(N - n0, tile_t::BN), 0, r1 - r0);
    const long long at = (long long)(L ? (int)blockIdx.y : e) * M * N;
    t.each([&](int m, int n, mh_f4 v) {
        const int c = N - n0 - n;
        if (m0 + m >= M || c <= 0) return;
        const long long i = at + (long long)(m0 + m) * N + n0 + n;
        if (L) mm_put4<MM_F32>(part + i, v, c);
        else mm_put4<TY>(static_cast<T*>(C_) + i, v, c);
    });
}

// out[e, i] = sum of part[s, i] over the group's slots, in their order: what ends a sum that was split over rows.
template <int TY>
__device__ __forceinline__ void mm_sum_body(const float* part, void* out_, const int* off, int R, int E, int L, long long n) {
    typedef typename mm_type<TY>::t T;
    const int e = blockIdx.y;
    const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 4;
    int s0 = 0, s1 = 0;
    if (!off) {
        s1 = (R + L - 1) / L;
    } else {
        int top = min(max(off[0], 0), R);               // as mm_slot
        for (int g = 0; g <= e; ++g) {
            const int hi = max(top, min(off[g + 1], R));
            s0 = s1;
            s1 += (hi - top + L - 1) / L;
            top = hi;
        }
    }
    if (i >= n) return;
    const int c = (int)min((long long)4, n - i);
    mh_f4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; ++s) v += mm_get4<MM_F32>(part + (long long)s * n + i, c);
    mm_put4<TY>(static_cast<T*>(out_) + (long long)e * n + i, v, c);
}

// p = g act'(a) in the type (P NULL: not stored, slope NULL: act' = 1) and the slots' sums of its columns in float32, before
// rounding, into part [slots, N] (NULL: none).  A workgroup takes a slot of L rows and 256 columns, 64 threads of four
// columns each by four rows at a time.
template <int TY>
__device__ __forceinline__ void mm_slope_body(const void* g_, const void* slope_, void* P_, float* part, const int* off,
                                              long long ldg, int R, int N, int E, int L) {
    typedef typename mm_type<TY>::t T;
    __shared__ mh_f4 sums[4][64];
    int e, r0, r1;
    if (!mm_slot(off, E, R, L, blockIdx.x, e, r0, r1)) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = blockIdx.y * 256 + 4 * lane, c = N - n;
    mh_f4 s = {0.f, 0.f, 0.f, 0.f};
    if (c > 0) {
        for (int r = r0 + w; r < r1; r += 4) {
            mh_f4 v = mm_get4<TY>(static_cast<const T*>(g_) + (long long)r * ldg + n, c);
            const long long at = (long long)r * N + n;
            if (slope_) {
                if constexpr (TY == MM_F32) {
                    v *= mm_get4<MM_F32>(static_cast<const float*>(slope_) + at, c);
                } else {
                    const unsigned short* q = static_cast<const unsigned short*>(slope_) + at;
                    mh_u2 k = {0u, 0u};
                    if (c >= 4) {
                        k = *reinterpret_cast<const mh_u2x*>(q);
                    } else {
                        k.x = q[0] | (c > 1 ? (unsigned)q[1] << 16 : 0u);
                        k.y = c > 2 ? q[2] : 0u;
                    }
                    v *= mh_f4{mm_slope_value(k.x & 0xFFFFu), mm_slope_value(k.x >> 16), mm_slope_value(k.y & 0xFFFFu),
                               mm_slope_value(k.y >> 16)};
                }
            }
            if (P_) mm_put4<TY>(static_cast<T*>(P_) + at, v, c);
            s += v;
        }
    }
    if (!part) return;
    sums[w][lane] = s;
    __syncthreads();
    if (w == 0 && c > 0) {
        s += sums[1][lane];
        s += sums[2][lane];
        s += sums[3][lane];
        mm_put4<MM_F32>(part + (long long)blockIdx.x * N + n, s, c);
    }
}
