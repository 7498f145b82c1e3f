// mh_halves.h — float32 matrix products as three float16 ones, prepended with mh_device.h and mh_matmul.h.
//
// A row (or column) of values times a power of two s that brings its largest to [2^14, 2^15) is, value by value, hi + 2^-12 lo
// with hi and lo float16: hi the nearest, lo the nearest to 2^12 times what is left.  a b = (hi_a + 2^-12 lo_a)
// (hi_b + 2^-12 lo_b) / (s_a s_b), where lo_a lo_b, below 2^-22 of |a b|, is left out: three products on the matrix cores where
// three bf16 parts need six, at the price of a pass that writes the halves (s must not change along the contraction, so one s
// per row of an operand that is contiguous along it, one per column and group of an operand whose rows are contracted).  Both
// forms keep the halves next to each other, as matrices of 16-bit values whose contraction is twice as long, which the tiles of
// mh_matmul.h load as they are:
//   rows    [R][Kp / 32][2][32]    32 hi, their 32 lo, ...; Kp = K rounded up to 32, zeros behind K
//   columns [R][2][Cp]             a row of hi, its row of lo; Cp = C rounded up to 8
//
// What the halves hold.  A value of at least 2^-14 after scaling is off by at most 2^-23 of itself, a smaller one by at most
// 2^-37.  So where both operands' values other than zero lie within 2^28 of their row's (column's) largest, a product is off by at
// most 2^-21 of |a b|, before what float32 sums add.  A row with a smaller value is `wide`: its results are off by up to
// K 2^-20 more in the units of the scaled sums, which is below K 2^-24 of any sum of at least 16 and so no more than a float32
// sum of K products may be off by.  What is left, results of a wide row or column below 16 (of largest products of 2^28 and
// more: one in 10^8 of random ones) and those of rows and columns with an infinity or NaN, are marked by row of the result,
// and hv_again computes the tiles that hold a marked one as the direct kernels do.
#pragma once

// What is known of a row's or column's values, a word: the exponent field of the largest, from bit 8 on 255 minus that of the
// smallest but zero (277 for subnormal ones; 0: zeros only), and
#define HV_AGAIN 0x40000000u        // a result of this row is to be computed again
#define HV_ODD 0x80000000u          // it holds an infinity or NaN
#define HV_LARGEST 0xFFu
#define HV_SMALLEST 0x1FF00u

__device__ __forceinline__ unsigned hv_word(float v) {
    const unsigned b = __float_as_uint(v) & 0x7FFFFFFFu, e = b >> 23;
    return b == 0u ? 0u : e == 255u ? HV_ODD : e | (e ? 255u - e : 277u) << 8;
}

// of two sets of values
__device__ __forceinline__ unsigned hv_join(unsigned a, unsigned b) {
    return max(a & HV_LARGEST, b & HV_LARGEST) | max(a & HV_SMALLEST, b & HV_SMALLEST) | ((a | b) & HV_ODD);
}

// exponent of s: 126 at most, beyond which float32 has no s
__device__ __forceinline__ int hv_shift(unsigned word) { return min(141 - (int)(word & HV_LARGEST), 126); }

// whether a value other than zero is below 2^-14 after scaling
__device__ __forceinline__ bool hv_wide(unsigned word) { return (int)((word & HV_SMALLEST) >> 8) > 142 + hv_shift(word); }

__device__ __forceinline__ void hv_split(float v, int shift, unsigned short& hi, unsigned short& lo) {
    const float t = __builtin_ldexpf(v, shift);
    const _Float16 h = (_Float16)t;
    const _Float16 l = (_Float16)((t - (float)h) * 4096.f);
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

// Rows: a wave each; the second reading of a row comes from the caches.  word [R + 1]: the last, whether anything is to be computed
// again, zero here.  Bound by its bytes: 20,000 rows of 1,024 in 39 us, 4.2 TB/s.
extern "C" __global__ __launch_bounds__(256) void hv_rows(const float* __restrict__ x, unsigned short* __restrict__ y,
                                                          unsigned* __restrict__ word, long long ld, int R, int K) {
    if (blockIdx.x == 0 && threadIdx.x == 0) word[R] = 0u;
    const int lane = threadIdx.x & 63, Kp = (K + 31) / 32 * 32;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    const float* p = x + r * ld;
    unsigned m = 0;
    for (int k = 4 * lane; k < K; k += 256) {
        const mh_f4 v = mm_get4<MM_F32>(p + k, K - k);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = hv_join(m, hv_word(v[j]));
    }
#pragma unroll
    for (int d = 1; d < MH_WAVE; d <<= 1) m = hv_join(m, (unsigned)__shfl_xor((int)m, d, MH_WAVE));
    if (lane == 0) word[r] = m;
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

// Columns, first pass: of each group's columns, the words in two arrays (zero before) whose largest values atomics can find: peak
// [E, C] the largest's exponents, mark [E, C] the smallest's and the odd ones' bit.  A workgroup for a piece of rows and 256
// columns.  The largest of integers does not depend on the order of the atomics.  Bound, with the second pass, by their bytes: 12
// a value, 1,024 x 1,024 weights 5.2 and 5.6 us.
extern "C" __global__ __launch_bounds__(256) void hv_peaks(const float* __restrict__ x, unsigned* __restrict__ peak,
                                                           unsigned* __restrict__ mark, const int* __restrict__ off,
                                                           long long ld, int R, int C, int E, int G, int L, int slots) {
    __shared__ unsigned best[4][64][4];
    int e, r0, r1;
    const int c0 = blockIdx.x / slots * 256;
    if (!hv_slot(off, E, R, G, L, blockIdx.x % slots, e, r0, r1)) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = c0 + 4 * lane;
    unsigned m[4] = {0u, 0u, 0u, 0u};
    if (c < C) {
#pragma unroll 4
        for (int r = r0 + w; r < r1; r += 4) {
            const mh_f4 v = mm_get4<MM_F32>(x + (long long)r * ld + c, C - c);
#pragma unroll
            for (int j = 0; j < 4; ++j) m[j] = hv_join(m[j], hv_word(v[j]));
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) best[w][lane][j] = m[j];
    __syncthreads();
    const int i = c0 + threadIdx.x;                      // a column a thread from here on
    if (i >= C) return;
    unsigned b = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) b = hv_join(b, best[k][threadIdx.x >> 2][threadIdx.x & 3]);
    atomicMax(&peak[(long long)e * C + i], b & HV_LARGEST);
    atomicMax(&mark[(long long)e * C + i], b & (HV_SMALLEST | HV_ODD));
}

// Columns, second pass: the halves.
extern "C" __global__ __launch_bounds__(256) void hv_columns(const float* __restrict__ x, unsigned short* __restrict__ y,
                                                             const unsigned* __restrict__ peak, const int* __restrict__ off,
                                                             long long ld, int R, int C, int E, int G, int L, int slots) {
    int e, r0, r1;
    if (!hv_slot(off, E, R, G, L, blockIdx.x % slots, e, r0, r1)) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x / slots * 256 + 4 * lane, Cp = (C + 7) / 8 * 8;
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

// The word of row or column i: one array, or (columns) two.
__device__ __forceinline__ unsigned hv_read(const unsigned* peak, const unsigned* mark, long long i) {
    return peak[i] | (mark ? mark[i] : 0u);
}

// A finished tile whose sums stand for sums times 2^(row's shift + column's): what mm_store_tile takes.
template <typename tile_t>
struct hv_result {
    static constexpr int ROWS = tile_t::ROWS, COLS = tile_t::COLS;
    const tile_t& t;
    const int rows, cols;
    unsigned a[ROWS];
    mh_u4 b[COLS];
    __device__ __forceinline__ static int row(int i) { return tile_t::row(i); }
    __device__ __forceinline__ static int column(int j) { return tile_t::column(j); }
    // words of the tile's rows and columns
    __device__ __forceinline__ hv_result(const tile_t& tile, const unsigned* pa, const unsigned* ma, int rows, const unsigned* pb,
                                         const unsigned* mb, int cols)
        : t(tile), rows(rows), cols(cols) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) a[i] = hv_read(pa, ma, min(row(i), rows - 1));
#pragma unroll
        for (int j = 0; j < COLS; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) b[j][c] = hv_read(pb, mb, min(column(j) + c, cols - 1));
    }
    __device__ __forceinline__ mh_f4 value(int i, int j) const {
        mh_f4 v = t.value(i, j);
        const int s = hv_shift(a[i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = __builtin_ldexpf(v[c], -(s + hv_shift(b[j][c])));
        return v;
    }
    // Marks the rows with results that the halves do not hold, in the words' array that keeps the smallest exponents (`at`: where
    // the tile's rows begin), and sets *any where there are such or odd rows or columns.  Workgroups of the same rows store the
    // same word.  Rows and columns of zeros alone give zeros, which are right.
    template <bool SPLIT>
    __device__ __forceinline__ void mark(unsigned* at, unsigned* any) const {
        unsigned some = 0u;
#pragma unroll
        for (int j = 0; j < COLS; ++j) some |= b[j].x | b[j].y | b[j].z | b[j].w;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const bool wide = hv_wide(a[i]);
            bool again = false;
            some |= a[i];
#pragma unroll
            for (int j = 0; j < COLS; ++j) {
                const mh_f4 v = t.value(i, j);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    again |= __builtin_fabsf(v[c]) < 16.f && (wide || hv_wide(b[j][c])) && (b[j][c] & HV_SMALLEST) &&
                             column(j) + c < cols;
            }
            if (again && row(i) < rows && (a[i] & HV_SMALLEST)) {
                at[row(i)] = (SPLIT ? a[i] & (HV_SMALLEST | HV_ODD) : a[i]) | HV_AGAIN;
                some = HV_ODD;
            }
        }
        if (some & HV_ODD) *any = 1u;
    }
};

// mm_rows_body on halves: A rows [R][Kp / 32][2][32] with their words pa [R + 1]; B either rows, [E][N][Kp / 32][2][32] with words
// pb [E][N], or (BS) columns of K contracted rows, [E][K][2][Np] with pb and mb [E][N].
// Bound by the matrix cores: 20,000 x 1,024 x 1,024 in 133 us, 950 TFLOP/s of float16 products (three rounds of workgroups where
// 2.45 would do), the cores busy 51 % of it.
template <bool BS, int ACT, typename tile_t>
__device__ __forceinline__ void hv_rows_body(const unsigned short* A, const unsigned short* B, float* C0, const float* bias,
                                             const float* res, float* slope, const int* off, unsigned* pa,
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
    const hv_result<tile_t> r(t, pa + r0, nullptr, rows, pb + col, mb ? mb + col : nullptr, cols);
    r.template mark<false>(pa + r0, pa + R);
    bias = bias ? bias + (long long)e * N : nullptr;
    if (n0 + tile_t::BN <= N) mm_store_tile<MM_F32, ACT, true>(r, r0, rows, n0, N, bias, res, ldr, slope, C0);
    else mm_store_tile<MM_F32, ACT, false>(r, r0, rows, n0, N, bias, res, ldr, slope, C0);
}

// mm_outer_body on halves: A columns [R][2][Mp], B columns [R][2][Np], their words [E][M], ma with one more behind, and [E][N].
template <typename tile_t>
__device__ __forceinline__ void hv_outer_body(const unsigned short* A, const unsigned short* B, float* C0, float* part,
                                              const int* off, const unsigned* pa, unsigned* ma, const unsigned* pb,
                                              const unsigned* mb, int R, int M, int N, int E, int L) {
    __shared__ mh_u4 lds[tile_t::LDS];
    const int NT = (N + tile_t::BN - 1) / tile_t::BN, MT = (M + tile_t::BM - 1) / tile_t::BM, y = blockIdx.x / (MT * NT);
    const int Mp = (M + 7) / 8 * 8, Np = (N + 7) / 8 * 8;
    int mt, nt, e = 0, r0 = 0, r1 = R;
    mm_tile_of(blockIdx.x % (MT * NT), MT * NT, MT, NT, mt, nt);
    if (L) {
        if (!mm_slot(off, E, R, L, y, e, r0, r1)) return;
    } else if (off) {
        mm_by_length(off, E, R, y, e, r0, r1);
    }
    const int m0 = mt * tile_t::BM, n0 = nt * tile_t::BN, rows = min(M - m0, tile_t::BM), cols = min(N - n0, tile_t::BN);
    const unsigned short *a = A + (long long)r0 * 2 * Mp + m0, *b = B + (long long)r0 * 2 * Np + n0;
    const int ar = min(Mp - m0, tile_t::BM), br = min(Np - n0, tile_t::BN);
    tile_t t;
    t.run(lds, a, Mp, ar, b, Np, br, 0, 2 * (r1 - r0));
    float* C = (L ? part + (long long)y * M * N : C0 + (long long)e * M * N) + (long long)m0 * N + n0;
    const long long ra = (long long)e * M + m0, rb = (long long)e * N + n0;
    const hv_result<tile_t> r(t, pa + ra, ma + ra, rows, pb + rb, mb + rb, cols);
    r.template mark<true>(ma + ra, ma + (long long)E * M);
#pragma unroll
    for (int i = 0; i < tile_t::ROWS; ++i)
#pragma unroll
        for (int j = 0; j < tile_t::COLS; ++j)
            if (tile_t::row(i) < rows && tile_t::column(j) < cols)
                mm_put4<MM_F32>(C + (long long)tile_t::row(i) * N + tile_t::column(j), r.value(i, j),
                                cols - tile_t::column(j));
}

// Whether a tile's rows or columns hold a marked one: the workgroup's answer, and the barrier between two tiles' products.
struct hv_marked {
    const unsigned *pa, *ma, *pb, *mb;
    int M, N;                                            // words a group of rows (0: none) and of columns
    __device__ __forceinline__ bool operator()(int e, int m0, int rows, int n0, int cols) const {
        if (e < 0) return false;
        unsigned any = 0;
        for (int i = threadIdx.x; i < rows; i += blockDim.x) any |= hv_read(pa, ma, (long long)e * M + m0 + i);
        for (int i = threadIdx.x; i < cols; i += blockDim.x) any |= hv_read(pb, mb, (long long)e * N + n0 + i);
        return __syncthreads_or((any & (HV_AGAIN | HV_ODD)) != 0u);
    }
};

// After hv_rows_body: the tiles with marked results once more, by the direct kernel from the operands themselves.  Workgroups walk
// the `tiles` where there is anything to do (all of 20,000 x 1,024 x 1,024: 330 us); where not, as nearly always, this costs a
// launch and one load, 4 us.
template <bool BS, int ACT, typename tile_t>
__device__ __forceinline__ void hv_again_rows_body(const float* A, const float* B, float* C, const float* bias, const float* res,
                                                   float* slope, const int* off, const unsigned* pa, const unsigned* pb,
                                                   const unsigned* mb, long long lda, long long ldb, long long ldr, int R, int N,
                                                   int K, int E, int tiles) {
    if (!pa[R]) return;
    const hv_marked marked = {pa, nullptr, pb, mb, 0, N};
    for (int b = blockIdx.x; b < tiles; b += gridDim.x)
        mm_rows_body<MM_F32, BS, ACT, tile_t>(A, B, C, bias, res, slope, off, lda, ldb, ldr, R, N, K, E, b, tiles, marked);
}

// After hv_outer_body, of `blocks` tiles in all groups or slots.
template <typename tile_t>
__device__ __forceinline__ void hv_again_outer_body(const float* A, const float* B, float* C, float* part, const int* off,
                                                    const unsigned* pa, const unsigned* ma, const unsigned* pb, const unsigned* mb,
                                                    long long lda, long long ldb, int R, int M, int N, int E, int L, int blocks) {
    if (!ma[(long long)E * M]) return;
    const hv_marked marked = {pa, ma, pb, mb, M, N};
    for (int b = blockIdx.x; b < blocks; b += gridDim.x)
        mm_outer_body<MM_F32, tile_t>(A, B, C, part, off, lda, ldb, R, M, N, E, L, b, marked);
}
