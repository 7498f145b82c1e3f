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
    // the sixteen bytes as they lie in memory, and their values; STREAM: data that nothing reads again soon
    template <bool STREAM = false>
    __device__ __forceinline__ static mh_u4 raw(const typename mm_type<TY>::t* p, int n) {
        if (n >= V) {
            if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const mh_u4x*>(p));
            else return *reinterpret_cast<const mh_u4x*>(p);
        }
        mh_u4 w = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) {
                if constexpr (TY == MM_F32) w[j] = __float_as_uint(p[j]);
                else w[j / 2] |= (unsigned)p[j] << (16 * (j & 1));
            }
        return w;
    }
    __device__ __forceinline__ void set(mh_u4 w) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if constexpr (TY == MM_F32) v[j] = __uint_as_float(w[j]);
            else v[j] = mm_widen<TY>((unsigned short)(w[j / 2] >> (16 * (j & 1))));
        }
    }
    __device__ __forceinline__ void get(const typename mm_type<TY>::t* p, int n) { set(raw(p, n)); }
    template <bool STREAM = false>
    __device__ __forceinline__ void put(typename mm_type<TY>::t* p, int n) const {
        if (n >= V) {
            mh_u4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (TY == MM_F32) w[j] = __float_as_uint(v[j]);
                else w[j] = mm_round<TY>(v[2 * j]) | (unsigned)mm_round<TY>(v[2 * j + 1]) << 16;
            }
            if constexpr (STREAM) __builtin_nontemporal_store((mh_u4x)w, reinterpret_cast<mh_u4x*>(p));
            else *reinterpret_cast<mh_u4x*>(p) = w;
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

// act(a), and act'(a) in `slope`, from one exponential: relu (NaN stays NaN), silu(a) = a q with q = 1 / (1 + e^-a) and slope
// q + a q (1 - q), gelu(a) = a Phi(a) with Phi the normal distribution function and slope Phi + a e^(-a^2/2) / sqrt(2 pi).
// For 128 values a thread these are a large part of a tile's time (a call of expf and two divisions each were 190 of 316 us
// at 16,384 x 4,096 x 1,024 in bfloat16), so: the hardware's 2^x and 1/x (one ulp each), with the rounding error of
// a log2(e) carried along for float32, and for the 16-bit types erf by Abramowitz and Stegun 7.1.26, erfc(z) =
// poly(1 / (1 + p z)) e^(-z^2) to 1.5e-7, which shares the slope's exponential; float32 calls erff.
template <int TY>
__device__ __forceinline__ float mm_exp(float a) {
    const float t = a * 1.44269504f;
    const float e = __builtin_amdgcn_exp2f(t);
    if constexpr (TY != MM_F32) return e;
    // 2^r = 1 + r ln 2 for what rounding left out of t; nothing to add to 0 and infinity
    const float r = __builtin_fmaf(a, 1.44269504f, -t) + a * 1.92596298e-8f;
    return e > 0.f && e < __builtin_inff() ? __builtin_fmaf(e * r, 0.69314718f, e) : e;
}

template <int TY, int ACT>
__device__ __forceinline__ float mm_activate(float a, float& slope) {
    if constexpr (ACT == MM_RELU) {
        slope = a > 0.f ? 1.f : 0.f;
        return a < 0.f ? 0.f : a;
    } else if constexpr (ACT == MM_SILU) {
        const float q = __builtin_amdgcn_rcpf(1.f + mm_exp<TY>(-a)), y = a * q;
        slope = __builtin_fmaf(y, 1.f - q, q);
        return y;
    } else if constexpr (ACT == MM_GELU) {
        const float g = mm_exp<TY>(-0.5f * a * a);
        float phi;
        if constexpr (TY == MM_F32) {
            phi = 0.5f * (1.f + erff(a * 0.70710678f));
        } else {
            const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678f, __builtin_fabsf(a), 1.f));
            float p = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
            p = __builtin_fmaf(t, p, 1.421413741f);
            p = __builtin_fmaf(t, p, -0.284496736f);
            p = __builtin_fmaf(t, p, 0.254829592f);
            const float c = 0.5f * t * p * g;            // Phi(-|a|)
            phi = a < 0.f ? c : 1.f - c;
        }
        slope = __builtin_fmaf(a * 0.39894228f, g, phi);
        return a * phi;
    }
    slope = 1.f;
    return a;
}

// act'(a) as the forward keeps it for the backward: float32, or for the 16-bit types a code of 16 bits.  The slopes of all
// activations lie in [-0.13, 1.13], and behind a unit's tail they fall below any fixed step, so a magnitude is coded in even steps
// of 2^-15 from 2^-7 on (float16: 2^-6), and below in steps of its own binade's 256th (512th) part, down to 2^-54 (2^-29).  Off by
// at most 2^-16 and, above that end, by 2^-9 (2^-10) of the slope, whichever is less: half of what rounding the product p to bfloat16
// adds, at most twice that for float16.  0 and 1 are exact.  Magnitudes count up from code 0, those of negative slopes down from
// 65535; 0xC000, between the two, is NaN.  Coding them is nine operations a value: 160 us at 16,384 x 4,096 x 1,024 in bfloat16 with
// silu, 142 without slopes (even steps alone, which lose the tails, took 153; float32 slopes would be 134 MB more, written and read).
template <int TY>
struct mm_slope_code {
    static constexpr int BITS = TY == MM_F16 ? 9 : 8;                        // of a small magnitude's mantissa
    static constexpr float EDGE = TY == MM_F16 ? 0x1p-6f : 0x1p-7f;          // where the even steps begin, at code 12288
    static constexpr float DOWN = TY == MM_F16 ? 0x1p-97f : 0x1p-72f;        // brings it to a float32 whose upper bits are its code
    static constexpr float UP = TY == MM_F16 ? 0x1p97f : 0x1p72f;
    static constexpr float FIRST = 12288.f - EDGE * 32768.f;                 // the even steps' code of 0
    __device__ __forceinline__ static unsigned of(float slope) {
        const float s = __builtin_fminf(slope, (49152.f - FIRST) * 0x1p-15f);        // NaN: the larger number, whose code is 0xC000
        const float m = __builtin_fabsf(s);
        const unsigned fine = (__float_as_uint(m * DOWN) + (1u << (22 - BITS))) >> (23 - BITS);
        const unsigned even = __float_as_uint(__builtin_fmaf(m, 32768.f, 8388608.f + FIRST));       // in its lower half
        return ((m < EDGE ? fine : even) ^ (unsigned)((int)__float_as_uint(s) >> 31)) & 0xFFFFu;
    }
    __device__ __forceinline__ static float value(unsigned code) {
        const unsigned sign = code > 0xC000u ? 0x80000000u : 0u, m = sign ? code ^ 0xFFFFu : code;
        const float v = m < 12288u ? __uint_as_float(m << (23 - BITS)) * UP : ((float)(int)m - FIRST) * 0x1p-15f;
        return __uint_as_float(code == 0xC000u ? 0x7FC00000u : __float_as_uint(v) | sign);
    }
};
// two at a time, the first in the lower half
template <int TY>
__device__ __forceinline__ unsigned mm_slope_codes(float lo, float hi) {
    return mm_slope_code<TY>::of(lo) | mm_slope_code<TY>::of(hi) << 16;
}

// ------------------------------------------------------------------------------------------------ groups of rows
// Rows [0, R) in E groups, group e from off[e] to off[e + 1].  Offsets are clamped into [0, R] and to the largest before them:
// whatever they hold, groups are disjoint and lead nowhere out of the tensors, and every kernel takes the same rows for a
// group.  64 groups at a time are scanned across a wave, every lane of which calls.
struct mm_groups {
    const int* __restrict__ off;
    int E, R;
    int lead;                                            // rows before the first group
    int top;                                             // where the groups scanned so far end
    int lo, hi;                                          // this lane's group of the 64 scanned last (empty past the last)
    __device__ __forceinline__ mm_groups(const int* offsets, int groups, int rows) : off(offsets), E(groups), R(rows) {
        top = lead = min(max(off[0], 0), R);
    }
    __device__ __forceinline__ void scan(int g0) {
        const int lane = threadIdx.x & (MH_WAVE - 1);
        hi = max(top, min(off[min(g0 + lane, E - 1) + 1], R));
#pragma unroll
        for (int d = 1; d < MH_WAVE; d <<= 1) {
            const int t = __shfl_up(hi, d, MH_WAVE);
            if (lane >= d) hi = max(hi, t);
        }
        const int prev = __shfl_up(hi, 1, MH_WAVE);
        lo = lane ? prev : top;
        top = mh_bcast(hi, MH_WAVE - 1);
    }
};

// Each group is cut into pieces of L rows, and slot s is the s-th piece.  False past the last one; the rows of no group then
// follow as pieces with e = -1, those before the first group and those behind the last.  off NULL: one group of all rows.
// There are at most R / L + E pieces (R / L + E + 2 with those of no group); R + L < 2^31.
__device__ __forceinline__ bool mm_slot(const int* __restrict__ off, int E, int R, int L, int s, int& e, int& r0, int& r1) {
    if (!off) {
        e = 0;
        r0 = s * L;
        r1 = min(R, r0 + L);
        return r0 < R;
    }
    const int lane = threadIdx.x & (MH_WAVE - 1);
    mm_groups g(off, E, R);
    int base = 0;                                        // pieces before these 64 groups
    for (int g0 = 0; g0 < E; g0 += MH_WAVE) {
        g.scan(g0);
        const int n = (g.hi - g.lo + L - 1) / L;
        int inc = n;
#pragma unroll
        for (int d = 1; d < MH_WAVE; d <<= 1) {
            const int t = __shfl_up(inc, d, MH_WAVE);
            if (lane >= d) inc += t;
        }
        const int total = mh_bcast(inc, MH_WAVE - 1);
        if (s < base + total) {
            const int l = __ffsll((unsigned long long)__ballot(base + inc > s)) - 1;
            const int glo = mh_bcast(g.lo, l), ghi = mh_bcast(g.hi, l), before = mh_bcast(inc - n, l);
            e = g0 + l;
            r0 = glo + (s - base - before) * L;
            r1 = min(ghi, r0 + L);
            return true;
        }
        base += total;
    }
    e = -1;
    const int d = s - base, first = (g.lead + L - 1) / L;        // pieces before the first group
    if (d < first) {
        r0 = d * L;
        r1 = min(g.lead, r0 + L);
    } else {
        r0 = (int)min(g.top + (long long)(d - first) * L, (long long)R);
        r1 = min(R, r0 + L);
    }
    return false;
}

// The rows of the group that is k-th by length, longest first (up to 64 groups; more are taken as they come): workgroups start in
// the order of their index, and a long group that starts last is what all others wait for.  Every lane of a wave calls.
__device__ __forceinline__ void mm_by_length(const int* __restrict__ off, int E, int R, int k, int& e, int& r0, int& r1) {
    const int lane = threadIdx.x & (MH_WAVE - 1);
    mm_groups g(off, E, R);
    int l = k % MH_WAVE;
    for (int g0 = 0; g0 <= k - l; g0 += MH_WAVE) g.scan(g0);
    if (E <= MH_WAVE) {
        const int n = g.hi - g.lo;
        int rank = 0;
        for (int i = 0; i < E; ++i) {
            const int m = mh_bcast(n, i);
            rank += m > n || (m == n && i < lane) ? 1 : 0;
        }
        l = __ffsll((unsigned long long)__ballot(lane < E && rank == k)) - 1;
        k = l;
    }
    e = k;
    r0 = mh_bcast(g.lo, l);
    r1 = mh_bcast(g.hi, l);
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
// (lane % 16) and stores them at once.  The next tile's loads to registers are in flight during a tile's products; one buffer of
// LDS, because a second one costs workgroups their place (bfloat16, 64 x 64, dw of 8,001 x 1,023 x 2,049 in pieces: 145 us
// with one, 208 with two).
template <int TY, bool AS, bool BS, int WM, int WN, int FM, int FN, int BK>
struct mm_tile {
    typedef typename mm_type<TY>::t T;
    static constexpr int THREADS = 64 * WM * WN, BM = 16 * FM * WM, BN = 16 * FN * WN, OPR = BK / 8, ROWS = FM, COLS = FN;
    static constexpr bool WHOLE_STEPS = false;
    static constexpr int PLANES = TY == MM_F32 ? 3 : 1;
    static constexpr int TA = PLANES * BM * OPR, TB = PLANES * BN * OPR;      // octets of a buffer
    static constexpr int LDS = TA + TB;
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
        lb.store(lds + TA);
        __syncthreads();
        for (int k = kbeg; k < kend; k += BK) {
            const bool more = k + BK < kend;
            if (more) {
                la.load(k + BK, kend);
                lb.load(k + BK, kend);
            }
            products(lds, lds + TA);
            if (!more) break;
            __syncthreads();                            // every wave has read the tile
            la.store(lds);
            lb.store(lds + TA);
            __syncthreads();
        }
    }

    // D[row(i), column(j) .. + 3] within the tile
    __device__ __forceinline__ static int row(int i) { return ((threadIdx.x >> 6) / WN) * 16 * FM + (threadIdx.x & 15) + 16 * i; }
    __device__ __forceinline__ static int column(int j) {
        return ((threadIdx.x >> 6) % WN) * 16 * FN + 4 * (threadIdx.x >> 4 & 3) + 16 * j;
    }
    __device__ __forceinline__ mh_f4 value(int i, int j) const {
        mh_f4 v = acc[i][j];
        if constexpr (TY == MM_F32) {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = __builtin_isfinite(v[c]) ? v[c] + low[i][j][c] : v[c];
        }
        return v;
    }
};

// The same sums for 16-bit operands that come to LDS without passing through registers: 16-byte buffer loads straight into it,
// double-buffered.  An operand contiguous along k is laid out as above; a strided one keeps its rows of k, [k][ROWS], and its
// fragments are read by transposing LDS reads (four k of 16 rows at a time).  Sixteen rows of a fragment are 32 bytes of a
// row of k, and the 32-byte pieces of row k are exchanged by f(k) so that the rows which one read touches fall into different
// banks.  Every operand's row distance and address are multiples of 16 bytes, and so are its rows' lengths, or they are padded
// to that, with zeros where the contraction runs along them (the caller sees to it); a load past the rows' end repeats the
// last ones, and one past kend is out of the buffer's range and gives zeros.
typedef __attribute__((address_space(3))) void mm_lds_void;

__device__ __forceinline__ int mm_turn(int k) { return (k & 3) | (k >> 1 & 4); }
__device__ __forceinline__ unsigned mm_lds_at(const void* p) {
    return (unsigned)(unsigned long long)(const __attribute__((address_space(3))) void*)p;
}

// Pairs of transposing reads at LDS bytes at[c] and at[c] + STEP, complete at the end of the block.  Written out because the
// compiler's own form of them waits for all loads into LDS that are under way, those of the next tile too.
template <int STEP>
__device__ __forceinline__ void mm_read_turned(const unsigned (&at)[4], mh_u2 (&lo)[4], mh_u2 (&hi)[4]) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %4, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %6, %10 offset:%12\n\t"
        "ds_read_b64_tr_b16 %3, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(STEP)
        : "memory");
}
template <int STEP>
__device__ __forceinline__ void mm_read_turned(const unsigned (&at)[2], mh_u2 (&lo)[2], mh_u2 (&hi)[2]) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %2, %4 offset:%6\n\t"
        "ds_read_b64_tr_b16 %1, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(hi[0]), "=&v"(hi[1])
        : "v"(at[0]), "v"(at[1]), "n"(STEP)
        : "memory");
}
template <bool STRIDED, int ROWS, int BK, int THREADS, bool HALVES>
struct mm_mover {
    static constexpr int OPR = BK / 8, ITEMS = ROWS * OPR / THREADS;
    static_assert(ROWS * OPR % THREADS == 0, "a tile is a whole number of loads per thread");
    unsigned off[ITEMS];                                 // byte offset of each load from the tile's first element
    int at[ITEMS];                                       // its k within the tile

    __device__ __forceinline__ void init(long long ld, int rows) {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int s = threadIdx.x + j * THREADS;
            if constexpr (STRIDED) {
                const int k = s / (ROWS / 8), p = s % (ROWS / 8);
                const int c = ((p >> 1) ^ (mm_turn(HALVES ? k >> 1 : k) & (ROWS / 16 - 1))) * 16 + (p & 1) * 8;
                at[j] = k;
                off[j] = (unsigned)(k * ld + min(c, rows - 8)) * 2;
            } else {
                const int r = s / OPR, o = (s % OPR) ^ (r / (16 / OPR) & (OPR - 1));
                at[j] = 8 * o;
                off[j] = (unsigned)(min(r, rows - 1) * ld + 8 * o) * 2;
            }
        }
    }
    // `left`: the k that exist from the tile's first on
    __device__ __forceinline__ void issue(const unsigned short* p, int left, mh_u4* tile) const {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned short*>(p), 0, 0x7fffffff, 0x00020000);
        const int w = threadIdx.x & ~63;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (mm_lds_void*)(tile + w + j * THREADS), 16,
                                                     at[j] < left ? off[j] : 0x80000000u, 0, 0, 0);
    }
};

template <int TY, bool AS, bool BS, int WM, int WN, int FM, int FN, int BK, bool HALVES = false>
struct mm_fast_tile {
    typedef unsigned short T;
    static constexpr int THREADS = 64 * WM * WN, BM = 16 * FM * WM, BN = 16 * FN * WN, ROWS = FM, COLS = FN;
    static constexpr bool WHOLE_STEPS = true;
    static constexpr int TA = BM * BK / 8, TB = BN * BK / 8, LDS = 2 * (TA + TB);
    mh_f4 acc[FM][FN];
    mh_f4 low[HALVES ? FM : 1][HALVES ? FN : 1];         // the products with a lower half, which is kept times 2^12

    // Fragments of 16 rows each from row0 on at k 32 ks .. + 31: contiguous operands by 16-byte reads; strided ones by
    // transposing reads, where sixteen lanes read four k of 16 rows (lane i: four rows of k i / 4) and lane i receives the
    // four k of row i.
    template <bool STRIDED, int ROWS, int N>
    __device__ __forceinline__ static void fragments(mh_u4 (&f)[N], mh_u4* tile, int row0, int ks) {
        const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
        if constexpr (STRIDED) {
            const int k = (HALVES ? 0 : 32 * ks) + 8 * q + (i >> 2), r = HALVES ? 2 * k + ks : k;
            constexpr int G = N < 4 ? N : 4;
#pragma unroll
            for (int h = 0; h < N; h += G) {
                unsigned at[G];
                mh_u2 lo[G], hi[G];
#pragma unroll
                for (int c = 0; c < G; ++c)
                    at[c] = mm_lds_at(tile) + 2 * (r * ROWS + ((row0 / 16 + h + c) ^ (mm_turn(k) & (ROWS / 16 - 1))) * 16 + (i & 3) * 4);
                mm_read_turned<(HALVES ? 16 : 8) * ROWS>(at, lo, hi);
#pragma unroll
                for (int c = 0; c < G; ++c) f[h + c] = mh_u4{lo[c].x, lo[c].y, hi[c].x, hi[c].y};
            }
        } else {
#pragma unroll
            for (int c = 0; c < N; ++c) f[c] = tile[mm_place<BK / 8>(row0 + 16 * c + i, 4 * ks + q)];
        }
    }

    __device__ __forceinline__ void products(mh_u4* a, mh_u4* b) {
        const int wave = threadIdx.x >> 6, ra = (wave / WN) * 16 * FM, rb = (wave % WN) * 16 * FN;
        if constexpr (HALVES) {
            // upper times upper, upper times lower, lower times upper
            mh_u4 fa[FM], fb[2][FN];
            fragments<BS, BN, FN>(fb[0], b, rb, 0);
            fragments<BS, BN, FN>(fb[1], b, rb, 1);
            fragments<AS, BM, FM>(fa, a, ra, 0);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    acc[i][j] = mm_mfma<TY>(fb[0][j], fa[i], acc[i][j]);
                    low[i][j] = mm_mfma<TY>(fb[1][j], fa[i], low[i][j]);
                }
            fragments<AS, BM, FM>(fa, a, ra, 1);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) low[i][j] = mm_mfma<TY>(fb[0][j], fa[i], low[i][j]);
            return;
        }
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) {
            mh_u4 fa[FM], fb[FN];
            fragments<BS, BN, FN>(fb, b, rb, ks);
            fragments<AS, BM, FM>(fa, a, ra, ks);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mm_mfma<TY>(fb[j], fa[i], acc[i][j]);
        }
    }

    // The loads of the next tile (where `left` > 0) and this one's products.  The four places are distinct: without that the
    // compiler waits for the loads before it reads the tile that is there.
    __device__ __forceinline__ void step(const mm_mover<AS, BM, BK, THREADS, HALVES>& ma,
                                         const mm_mover<BS, BN, BK, THREADS, HALVES>& mb, const T* A, const T* B, int left,
                                         int bleft, mh_u4* __restrict__ a, mh_u4* __restrict__ b, mh_u4* __restrict__ an,
                                         mh_u4* __restrict__ bn) {
        if (left > 0) {
            ma.issue(A, left, an);
            mb.issue(B, bleft, bn);
        }
        products(a, b);
    }

    // `bend`: where B's k end, if before A's (whose padding is zeros); 0: with A's
    __device__ __forceinline__ void run(mh_u4* lds, const T* A, long long lda, int arows, const T* B, long long ldb, int brows,
                                        int kbeg, int kend, int bend = 0) {
        if (!bend) bend = kend;
        mm_mover<AS, BM, BK, THREADS, HALVES> ma;
        mm_mover<BS, BN, BK, THREADS, HALVES> mb;
        ma.init(lda, arows);
        mb.init(ldb, brows);
        const long long sa = AS ? lda : 1, sb = BS ? ldb : 1;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                acc[i][j] = mh_f4{0.f, 0.f, 0.f, 0.f};
                if constexpr (HALVES) low[i][j] = mh_f4{0.f, 0.f, 0.f, 0.f};
            }
        if (kbeg >= kend) return;                       // uniform over the workgroup
        mh_u4 *a0 = lds, *a1 = lds + TA, *b0 = lds + 2 * TA, *b1 = lds + 2 * TA + TB;
        ma.issue(A + kbeg * sa, kend - kbeg, a0);
        mb.issue(B + kbeg * sb, bend - kbeg, b0);
        for (int k = kbeg; k < kend; k += BK) {
            // the tile of this step is in LDS, and every wave is done with the other buffer
            __builtin_amdgcn_s_waitcnt(0x0F70);         // vmcnt(0)
            __syncthreads();
            step(ma, mb, A + (k + BK) * sa, B + (k + BK) * sb, kend - k - BK, bend - k - BK, a0, b0, a1, b1);
            mh_u4* t = a0;
            a0 = a1;
            a1 = t;
            t = b0;
            b0 = b1;
            b1 = t;
        }
    }

    __device__ __forceinline__ static int row(int i) { return ((threadIdx.x >> 6) / WN) * 16 * FM + (threadIdx.x & 15) + 16 * i; }
    __device__ __forceinline__ static int column(int j) {
        return ((threadIdx.x >> 6) % WN) * 16 * FN + 4 * (threadIdx.x >> 4 & 3) + 16 * j;
    }
    __device__ __forceinline__ mh_f4 value(int i, int j) const {
        if constexpr (HALVES) return acc[i][j] + low[i][j] * 0x1p-12f;
        else return acc[i][j];
    }
};

// The length of a strided operand's rows as a tile may load them: whole steps of 16 bytes where it goes straight to LDS (rows
// are padded to that; what the padding holds reaches only results that are not stored).
template <typename tile_t, bool STRIDED>
__device__ __forceinline__ int mm_wide(int n) { return STRIDED && tile_t::WHOLE_STEPS ? (n + 7) & ~7 : n; }

// The tile (mt, nt) of a block among MT x NT: bands of eight row tiles, walked column by column, in one contiguous range
// per XCD, so that blocks which share an L2 share operand tiles.
__device__ __forceinline__ void mm_tile_of(int b, int blocks, int MT, int NT, int& mt, int& nt) {
    const int l = mh_xcd_block(b, blocks), band = 8 * NT, first = l / band * 8, high = min(8, MT - first), i = l % band;
    mt = first + i % high;
    nt = i / high;
}

// What follows the sums v of four outputs, at element `at` of the result, of which `c` exist: activation with its slope kept
// where wanted, residual, one rounding (the bias is in v already).
template <int TY, int ACT>
__device__ __forceinline__ void mm_finish(mh_f4 v, long long at, int c, mh_f4 res, void* slope_, typename mm_type<TY>::t* C) {
    if constexpr (ACT != MM_NONE) {
        mh_f4 d;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float t;
            v[j] = mm_activate<TY, ACT>(v[j], t);
            d[j] = t;
        }
        if (slope_) {
            if constexpr (TY == MM_F32) {
                mm_put4<MM_F32>(static_cast<float*>(slope_) + at, d, c);
            } else {
                unsigned short* s = static_cast<unsigned short*>(slope_) + at;
                const mh_u2 w = {mm_slope_codes<TY>(d[0], d[1]), mm_slope_codes<TY>(d[2], d[3])};
                if (c >= 4)
                    *reinterpret_cast<mh_u2x*>(s) = w;
                else
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        if (j < c) s[j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
            }
        }
    }
    mm_put4<TY>(C + at, v + res, c);
}

// A tile's results to C at rows r0 .. + rows and columns n0 on.  The bias is loaded once for all rows, the residual a row of
// fragments at a time: loaded one by one between the activations they were 85 of 274 us (bias, 16,384 x 4,096 x 1,024 in
// bfloat16).  WHOLE: all columns of the tile exist.
template <int TY, int ACT, bool WHOLE, typename tile_t>
__device__ __forceinline__ void mm_store_tile(const tile_t& t, long long r0, int rows, int n0, int N,
                                              const typename mm_type<TY>::t* bias, const typename mm_type<TY>::t* res,
                                              long long ldr, void* slope, typename mm_type<TY>::t* C) {
    constexpr int FM = tile_t::ROWS, FN = tile_t::COLS;
    const mh_f4 zero = {0.f, 0.f, 0.f, 0.f};
    mh_f4 bv[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + tile_t::column(j), c = WHOLE ? 4 : N - n;
        bv[j] = bias && c > 0 ? mm_get4<TY>(bias + n, c) : zero;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = tile_t::row(i);
        if (m >= rows) continue;
        mh_f4 rv[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + tile_t::column(j), c = WHOLE ? 4 : N - n;
            rv[j] = res && c > 0 ? mm_get4<TY>(res + (r0 + m) * ldr + n, c) : zero;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + tile_t::column(j), c = WHOLE ? 4 : N - n;
            if (c > 0) mm_finish<TY, ACT>(t.value(i, j) + bv[j], (r0 + m) * N + n, c, rv[j], slope, C);
        }
    }
}

// The same for a whole-column tile of 16-bit results whose rows start at multiples of 16 bytes: a wave turns sixteen of its
// rows at a time in LDS, so that a store writes whole 128-byte lines of eight rows where the lanes' own eight bytes lie in
// 32-byte pieces of sixteen.
template <int TY, int ACT, typename tile_t>
__device__ __forceinline__ void mm_store_lines(const tile_t& t, mh_u4* lds, long long r0, int rows, int n0, int N,
                                               const unsigned short* bias, const unsigned short* res, long long ldr,
                                               unsigned short* slope, unsigned short* C) {
    constexpr int FM = tile_t::ROWS, FN = tile_t::COLS, W = 16 * FN, LD = W + 8, PER = 64 / (W / 8);
    static_assert(tile_t::THREADS / 64 * 2 * 16 * LD * 2 <= tile_t::LDS * 16, "the waves' places fit the tile's buffers");
    const int lane = threadIdx.x & 63, i16 = lane & 15, q = lane >> 4;
    unsigned short* y = reinterpret_cast<unsigned short*>(lds) + (threadIdx.x >> 6) * 2 * 16 * LD;
    unsigned short* d = y + 16 * LD;
    mh_f4 bv[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) bv[j] = bias ? mm_get4<TY>(bias + n0 + tile_t::column(j)) : mh_f4{0.f, 0.f, 0.f, 0.f};
    const int first = tile_t::row(0) - i16, left = n0 + tile_t::column(0) - 4 * q;      // the wave's corner
    __syncthreads();                                     // every wave is done with the tile's buffers
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = min(tile_t::row(i), rows - 1);
        mh_f4 rv[FN];
        if (res)
#pragma unroll
            for (int j = 0; j < FN; ++j) rv[j] = mm_get4<TY>(res + (r0 + m) * ldr + n0 + tile_t::column(j));
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            mh_f4 v = t.value(i, j) + bv[j], c;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float s;
                v[k] = mm_activate<TY, ACT>(v[k], s);
                c[k] = s;
            }
            const int at = i16 * LD + 16 * j + 4 * q;
            if (res) v += rv[j];
            *reinterpret_cast<mh_u2*>(y + at) = mh_u2{mm_round<TY>(v.x) | (unsigned)mm_round<TY>(v.y) << 16,
                                                      mm_round<TY>(v.z) | (unsigned)mm_round<TY>(v.w) << 16};
            if (ACT != MM_NONE && slope)
                *reinterpret_cast<mh_u2*>(d + at) = mh_u2{mm_slope_codes<TY>(c.x, c.y), mm_slope_codes<TY>(c.z, c.w)};
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < 16; s += PER) {
            const int r = s + lane / (W / 8), c = lane % (W / 8) * 8, m = first + 16 * i + r;
            if (m < rows) {
                const long long at = (r0 + m) * N + left + c;
                *reinterpret_cast<mh_u4*>(C + at) = *reinterpret_cast<const mh_u4*>(y + r * LD + c);
                if (ACT != MM_NONE && slope)             // not read before the backward: past the caches
                    __builtin_nontemporal_store(*reinterpret_cast<const mh_u4*>(d + r * LD + c),
                                                reinterpret_cast<mh_u4*>(slope + at));
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Every tile is wanted: what the bodies below ask before a tile's products (mh_halves.h asks otherwise).
struct mm_every {
    __device__ __forceinline__ bool operator()(int, int, int, int, int) const { return true; }
};

// Forward and input gradient: R rows of A [R, K] in groups, B the group's weights ([N, K], or [K, N] where BS), the
// epilogue v = sums + bias[e]; slope = act'(v); C = act(v) + res.  Rows of no group are written as zeros.  `b` of `blocks`
// tiles; wanted(e, first row, rows, first column, columns): whether to write it (e -1: rows of no group).
template <int TY, bool BS, int ACT, typename tile_t, typename wanted_t = mm_every>
__device__ __forceinline__ void mm_rows_body(const void* A_, const void* B_, void* C_, const void* bias_, const void* res_,
                                             void* slope_, const int* off, long long lda, long long ldb, long long ldr, int R, int N,
                                             int K, int E, int b = blockIdx.x, int blocks = gridDim.x,
                                             wanted_t wanted = wanted_t()) {
    typedef typename mm_type<TY>::t T;
    __shared__ mh_u4 lds[tile_t::LDS];
    const int NT = (N + tile_t::BN - 1) / tile_t::BN, MT = blocks / NT;
    int mt, nt, e, r0, r1;
    mm_tile_of(b, blocks, MT, NT, mt, nt);
    const bool live = mm_slot(off, E, R, tile_t::BM, mt, e, r0, r1);
    if (r0 >= R) return;
    const int n0 = nt * tile_t::BN, rows = r1 - r0;
    if (!wanted(e, r0, rows, n0, min(N - n0, tile_t::BN))) return;
    T* C = static_cast<T*>(C_) + (long long)r0 * N + n0;
    tile_t t;
    if (!live) {
        // rows without a group
        for (int i = threadIdx.x; i < rows * min(N - n0, tile_t::BN); i += tile_t::THREADS) {
            const int w = min(N - n0, tile_t::BN);
            C[(long long)(i / w) * N + i % w] = 0;
        }
        return;
    }
    const T* A = static_cast<const T*>(A_) + (long long)r0 * lda;
    const T* B = static_cast<const T*>(B_) + (BS ? (long long)e * K * ldb + n0 : ((long long)e * N + n0) * ldb);
    t.run(lds, A, lda, rows, B, ldb, min(mm_wide<tile_t, BS>(N) - n0, tile_t::BN), 0, K);
    const T* bias = bias_ ? static_cast<const T*>(bias_) + (long long)e * N : nullptr;
    const T* res = static_cast<const T*>(res_);
    if constexpr (TY != MM_F32) {
        if (n0 + tile_t::BN <= N && N % 8 == 0) {
            mm_store_lines<TY, ACT>(t, lds, r0, rows, n0, N, bias, res, ldr, static_cast<T*>(slope_), static_cast<T*>(C_));
            return;
        }
    }
    if (n0 + tile_t::BN <= N)
        mm_store_tile<TY, ACT, true>(t, r0, rows, n0, N, bias, res, ldr, slope_, static_cast<T*>(C_));
    else
        mm_store_tile<TY, ACT, false>(t, r0, rows, n0, N, bias, res, ldr, slope_, static_cast<T*>(C_));
}

// The forward for few rows: a workgroup takes 16 TM rows of a group and 16 columns, its WAVES waves share the contraction and
// add their sums through LDS in wave order.  Both operands go from memory to the matrix cores' registers: weights are read
// once and no tile of rows is worth staging.  Bound by the weights' bytes and by latency: a wave keeps four 128-byte
// pieces of 16 weight rows in flight.  One row of 1,024 to 4,096 in bfloat16 takes 4.1 us (8.4 MB, 2 TB/s: two trips to memory
// and a launch), eight rows of different ones of 64 experts of 1,024 to 2,048 9 us, one row of each of 64 groups of 1,024 to
// 4,096 105 us (5.1 TB/s).  float32 uses v_mfma_f32_16x16x4_f32 (k in the order 4 q + j of four steps).
template <int TY, int ACT, int TM, int WAVES>
__device__ __forceinline__ void mm_few_body(const void* A_, const void* B_, void* C_, const void* bias_, const void* res_,
                                            void* slope_, const int* off, long long lda, long long ldb, long long ldr, int R, int N,
                                            int K, int E) {
    typedef typename mm_type<TY>::t T;
    constexpr int V = TY == MM_F32 ? 4 : 8, STEP = 4 * V, BATCH = 4;
    __shared__ mh_f4 sums[WAVES][TM][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    const int NT = (N + 15) / 16, mt = blockIdx.x / NT, n0 = blockIdx.x % NT * 16;
    int e, r0, r1;
    const bool live = mm_slot(off, E, R, 16 * TM, mt, e, r0, r1);
    if (r0 >= R) return;
    const int rows = r1 - r0, cols = min(N - n0, 16);
    T* C = static_cast<T*>(C_);
    if (!live) {
        for (int j = threadIdx.x; j < rows * cols; j += 64 * WAVES) C[(long long)(r0 + j / cols) * N + n0 + j % cols] = 0;
        return;
    }
    const T* b = static_cast<const T*>(B_) + ((long long)e * N + n0 + min(i, cols - 1)) * ldb + V * q;
    const T* a[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t)
        a[t] = static_cast<const T*>(A_) + (long long)(r0 + min(16 * t + i, rows - 1)) * lda + V * q;
    mh_f4 acc[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) acc[t] = mh_f4{0.f, 0.f, 0.f, 0.f};
    auto product = [&](mh_u4 w, mh_u4 x, mh_f4 c) {
        if constexpr (TY == MM_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[j]), __uint_as_float(x[j]), c, 0, 0, 0);
            return c;
        } else {
            return mm_mfma<TY>(w, x, c);
        }
    };
    // pairs of steps (128 bytes of a row), wave by wave
    const int pairs = K / (2 * STEP);
    int p = wave;
    for (; p + (BATCH - 1) * WAVES < pairs; p += BATCH * WAVES) {
        mh_u4 w[2 * BATCH], x[TM][2 * BATCH];
#pragma unroll
        for (int u = 0; u < 2 * BATCH; ++u)
            w[u] = *reinterpret_cast<const mh_u4x*>(b + ((p + u / 2 * WAVES) * 2 + u % 2) * STEP);
#pragma unroll
        for (int t = 0; t < TM; ++t)
#pragma unroll
            for (int u = 0; u < 2 * BATCH; ++u)
                x[t][u] = *reinterpret_cast<const mh_u4x*>(a[t] + ((p + u / 2 * WAVES) * 2 + u % 2) * STEP);
#pragma unroll
        for (int u = 0; u < 2 * BATCH; ++u)
#pragma unroll
            for (int t = 0; t < TM; ++t) acc[t] = product(w[u], x[t][u], acc[t]);
    }
    for (; p < pairs; p += WAVES)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const mh_u4 w = *reinterpret_cast<const mh_u4x*>(b + (p * 2 + u) * STEP);
#pragma unroll
            for (int t = 0; t < TM; ++t)
                acc[t] = product(w, *reinterpret_cast<const mh_u4x*>(a[t] + (p * 2 + u) * STEP), acc[t]);
        }
    // what a pair does not fill, by the last wave; both operands are zero past K
    if (wave == WAVES - 1)
        for (int k = pairs * 2 * STEP; k < K; k += STEP) {
            const int left = K - k - V * q;
            auto get = [&](const T* s) {
                if (left >= V) return (mh_u4) * reinterpret_cast<const mh_u4x*>(s);
                mh_u4 v = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) {
                        if constexpr (TY == MM_F32) v[j] = __float_as_uint(s[j]);
                        else v[j / 2] |= (unsigned)s[j] << (16 * (j & 1));
                    }
                return v;
            };
            const mh_u4 w = get(b + k);
#pragma unroll
            for (int t = 0; t < TM; ++t) acc[t] = product(w, get(a[t] + k), acc[t]);
        }
#pragma unroll
    for (int t = 0; t < TM; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < TM; t += WAVES) {
        mh_f4 v = sums[0][t][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += sums[k][t][lane];
        const int c = cols - 4 * q, n = n0 + 4 * q;
        const long long r = (long long)r0 + 16 * t + i;
        if (16 * t + i < rows && c > 0) {
            if (bias_) v += mm_get4<TY>(static_cast<const T*>(bias_) + (long long)e * N + n, c);
            const mh_f4 res = res_ ? mm_get4<TY>(static_cast<const T*>(res_) + r * ldr + n, c) : mh_f4{0.f, 0.f, 0.f, 0.f};
            mm_finish<TY, ACT>(v, r * N + n, c, res, slope_, C);
        }
    }
}

// Weight gradients: D[e] [M, N] = sum over the group's rows of A[r, m] B[r, n] (A = p [R, M], B = x [R, N]).  Blocks count the
// tiles of the result, and these for one y after the other: the group (L 0: all its rows; none give zeros), or a slot of at most L
// of its rows whose sums go to part[slot] in float32.  wanted as in mm_rows_body, of the result's rows and columns.
// Bound as the other products; 16,384 rows of 4,096 by 1,024 in bfloat16 in four pieces take 140 us and 10 for their sum
// (980 TFLOP/s), eight groups of 2,048 rows of 2,048 by 1,024 whole 75 us.
template <int TY, typename tile_t, typename wanted_t = mm_every>
__device__ __forceinline__ void mm_outer_body(const void* A_, const void* B_, void* C_, float* part, const int* off,
                                              long long lda, long long ldb, int R, int M, int N, int E, int L,
                                              unsigned block = blockIdx.x, wanted_t wanted = wanted_t()) {
    typedef typename mm_type<TY>::t T;
    __shared__ mh_u4 lds[tile_t::LDS];
    const int NT = (N + tile_t::BN - 1) / tile_t::BN, MT = (M + tile_t::BM - 1) / tile_t::BM, y = block / (MT * NT);
    int mt, nt, e = 0, r0 = 0, r1 = R;
    mm_tile_of(block % (MT * NT), MT * NT, MT, NT, mt, nt);
    if (L) {
        if (!mm_slot(off, E, R, L, y, e, r0, r1)) return;
    } else if (off) {
        mm_by_length(off, E, R, y, e, r0, r1);
    }
    const int m0 = mt * tile_t::BM, n0 = nt * tile_t::BN;
    if (!wanted(e, m0, min(M - m0, tile_t::BM), n0, min(N - n0, tile_t::BN))) return;
    tile_t t;
    t.run(lds, static_cast<const T*>(A_) + (long long)r0 * lda + m0, lda, min(mm_wide<tile_t, true>(M) - m0, tile_t::BM),
          static_cast<const T*>(B_) + (long long)r0 * ldb + n0, ldb, min(mm_wide<tile_t, true>(N) - n0, tile_t::BN), 0,
          r1 - r0);
    const long long at = (long long)(L ? y : e) * M * N;
#pragma unroll
    for (int i = 0; i < tile_t::ROWS; ++i)
#pragma unroll
        for (int j = 0; j < tile_t::COLS; ++j) {
            const int m = m0 + tile_t::row(i), n = n0 + tile_t::column(j), c = N - n;
            if (m >= M || c <= 0) continue;
            const long long k = at + (long long)m * N + n;
            if (L) mm_put4<MM_F32>(part + k, t.value(i, j), c);
            else mm_put4<TY>(static_cast<T*>(C_) + k, t.value(i, j), c);
        }
}

// The slots of group e, as mm_slot numbers them.  Every lane of a wave calls.
__device__ __forceinline__ void mm_slots_of(const int* __restrict__ off, int E, int R, int L, int e, int& s0, int& s1) {
    s0 = 0;
    s1 = (R + L - 1) / L;
    if (!off) return;
    mm_groups g(off, E, R);
    int base = 0;
    for (int g0 = 0;; g0 += MH_WAVE) {
        g.scan(g0);
        const int l = e - g0, n = (g.hi - g.lo + L - 1) / L;
        int inc = n;
#pragma unroll
        for (int d = 1; d < MH_WAVE; d <<= 1) {
            const int t = __shfl_up(inc, d, MH_WAVE);
            if ((int)(threadIdx.x & (MH_WAVE - 1)) >= d) inc += t;
        }
        if (l < MH_WAVE) {
            s1 = base + mh_bcast(inc, l);
            s0 = s1 - mh_bcast(n, l);
            return;
        }
        base += mh_bcast(inc, MH_WAVE - 1);
    }
}

// out[e, i] = sum of part[s, i] over the group's slots in a fixed order: what ends a sum that was split over rows.  2^lg waves
// share a column's slots (wave w takes every 2^lg-th) and are added in wave order, so that few columns of many slots are
// not one wave's chain of loads; 1024 threads, four columns a lane.  Bound by its bytes: 4 slots of 4,096 x 1,024 in 10 us, 512
// slots of 6,144 columns in 5.
template <int TY>
__device__ __forceinline__ void mm_sum_body(const float* part, void* out_, const int* off, int R, int E, int L, int lg,
                                            long long n) {
    typedef typename mm_type<TY>::t T;
    __shared__ mh_f4 sums[16][64];
    const long long columns = 256 * (16 >> lg), per = (n + columns - 1) / columns;       // blocks of a group
    const int e = (int)(blockIdx.x / per), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = wave & ((1 << lg) - 1);
    const long long i = blockIdx.x % per * columns + (wave >> lg) * 256 + 4 * lane;
    int s0, s1;
    mm_slots_of(off, E, R, L, e, s0, s1);
    const int c = (int)max((long long)0, min((long long)4, n - i));
    mh_f4 v = {0.f, 0.f, 0.f, 0.f};
    if (c >= 4) {
#pragma unroll 8
        for (int s = s0 + w; s < s1; s += 1 << lg) v += mm_get4<MM_F32>(part + (long long)s * n + i);
    } else if (c > 0) {
        for (int s = s0 + w; s < s1; s += 1 << lg) v += mm_get4<MM_F32>(part + (long long)s * n + i, c);
    }
    if (lg) {
        sums[wave][lane] = v;
        __syncthreads();
        if (w) return;
        for (int k = 1; k < 1 << lg; ++k) v += sums[wave + k][lane];
    }
    if (c > 0) mm_put4<TY>(static_cast<T*>(out_) + (long long)e * n + i, v, c);
}

// p = g act'(a) in the type (P NULL: not stored, slope NULL: act' = 1), rows ldp >= N apart with zeros behind N, and the sums of
// its columns in float32, before rounding: into part [slots, N] for each slot of L rows, or, where one slot holds all rows,
// rounded into db (both NULL: none).  For 16-bit types p is rounded once here, as the matrix products take it: the error of a
// gradient is then that of a product of rounded operands.  A workgroup takes a slot and 256 columns (blocks count the slots of
// the first 256, then of the next), 64 threads of four columns each by four rows at a time.  Bound by its bytes; the slope is read for the last time, past the caches: 69 us at
// 16,384 x 4,096 bfloat16, 5.8 TB/s (81 as an ordinary read).
template <int TY>
__device__ __forceinline__ void mm_slope_body(const void* g_, const void* slope_, void* P_, float* part, void* db, const int* off,
                                              long long ldg, long long ldp, int R, int N, int E, int L, int slots) {
    typedef typename mm_type<TY>::t T;
    __shared__ mh_f4 sums[4][64];
    int e, r0, r1;
    const int slot = blockIdx.x % slots;
    if (!mm_slot(off, E, R, L, slot, e, r0, r1) && !db) return;            // db without rows: zeros
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = blockIdx.x / slots * 256 + 4 * lane, c = N - n;
    const T* g = static_cast<const T*>(g_) + n;
    T* P = static_cast<T*>(P_);
    mh_f4 s = {0.f, 0.f, 0.f, 0.f};
    auto times = [&](mh_f4 v, mh_u4 d) {                 // the slope as it was loaded
        if constexpr (TY == MM_F32) {
            return v * __builtin_bit_cast(mh_f4, d);
        } else {
            typedef mm_slope_code<TY> code;
            return v * mh_f4{code::value(d.x & 0xFFFFu), code::value(d.x >> 16), code::value(d.y & 0xFFFFu),
                             code::value(d.y >> 16)};
        }
    };
    if (c >= 4) {
#pragma unroll 4
        for (int r = r0 + w; r < r1; r += 4) {
            mh_f4 v = mm_get4<TY>(g + (long long)r * ldg);
            const long long at = (long long)r * N + n;
            if (slope_) {
                if constexpr (TY == MM_F32) {
                    v = times(v, __builtin_nontemporal_load(
                                     reinterpret_cast<const mh_u4x*>(static_cast<const float*>(slope_) + at)));
                } else {
                    const mh_u2 d = __builtin_nontemporal_load(
                        reinterpret_cast<const mh_u2x*>(static_cast<const unsigned short*>(slope_) + at));
                    v = times(v, mh_u4{d.x, d.y, 0u, 0u});
                }
            }
            if (P) mm_put4<TY>(P + r * ldp + n, v);
            s += v;
        }
    } else if (c > 0) {
        for (int r = r0 + w; r < r1; r += 4) {
            mh_f4 v = mm_get4<TY>(g + (long long)r * ldg, c);
            const long long at = (long long)r * N + n;
            if (slope_) {
                mh_u4 d = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < 4; ++j) {            // behind the row: v is zero there, and the slope too
                    if constexpr (TY == MM_F32) d[j] = j < c ? static_cast<const unsigned*>(slope_)[at + j] : 0u;
                    else d[j / 2] |= (j < c ? static_cast<const unsigned short*>(slope_)[at + j] : 0u) << (16 * (j & 1));
                }
                v = times(v, d);
            }
            if (P) mm_put4<TY>(P + r * ldp + n, v, (int)min((long long)4, ldp - n));
            s += v;
        }
    } else if (P && n < ldp) {
        for (int r = r0 + w; r < r1; r += 4) mm_put4<TY>(P + r * ldp + n, s, (int)min((long long)4, ldp - n));
    }
    if (!part && !db) return;
    sums[w][lane] = s;
    __syncthreads();
    if (w == 0 && c > 0) {
        s += sums[1][lane];
        s += sums[2][lane];
        s += sums[3][lane];
        if (db) mm_put4<TY>(static_cast<T*>(db) + n, s, c);
        else mm_put4<MM_F32>(part + (long long)slot * N + n, s, c);
    }
}

// y [R, Kp] = x [R, K] with zeros behind K: rows of 16-bit values at whole steps of 16 bytes.  A thread copies one step;
// bound by its bytes, about 4.5 TB/s where they are many.
template <int TY>
__device__ __forceinline__ void mm_pad_body(const void* x, void* y, long long ld, int R, int K, int Kp) {
    typedef typename mm_type<TY>::t T;
    const int steps = Kp / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, r = i / steps;
    const int k = (int)(i % steps) * 8;
    if (r < R)
        *reinterpret_cast<mh_u4*>(static_cast<T*>(y) + r * Kp + k) =
            mm_vec<TY>::raw(static_cast<const T*>(x) + r * ld + k, K - k);
}
