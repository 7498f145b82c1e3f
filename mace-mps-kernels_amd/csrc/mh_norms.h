// mh_norms.h — norms before and after a block, fused with its gate and residual scale; prepended with mh_device.h and
// mh_matmul.h.
//
// With N(v) = (v - mean v) / sqrt(var v + eps) (LAYER) or v / sqrt(mean v^2 + eps), per row of C values:
//   u = N(y),  h = x + s gate u wp,  v = N(h),  n = v wn                       (s, gate, wp, wn: 1 where absent)
// and backward, with q = gn wn and M the mean over the row:
//   dh = gh + r_h (q - v M(q v) [- M(q)]),  dx = dh,  dwn = sum_t gn v
//   e = dh s gate wp,  dy = r_y (e - u M(e u) [- M(e)]),  ds = sum dh gate u wp,  dwp = sum dh s gate u,
//   dgate = dh s u wp (summed over the row for a gate of one value per row).
// A row's values stay in registers between the sums that they need (one read of each input), all sums are float32.
#pragma once

// A row of up to TPR NV V values, thread l holding vectors l, l + TPR, ...; TPR up to 64: a part of a wave (256 / TPR rows a
// workgroup), more: the workgroup.
__device__ constexpr int nm_waves(int tpr) { return tpr > MH_WAVE ? tpr / MH_WAVE : 1; }
__device__ constexpr int nm_rows(int tpr) { return tpr > MH_WAVE ? 1 : 256 / tpr; }
template <int TY, int TPR, int NV>
struct nm_row {
    typedef typename mm_type<TY>::t T;
    static constexpr int V = mm_vec<TY>::V;
    mm_vec<TY> r[NV];
    __device__ __forceinline__ void get(const T* p, int C, int l) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + i * TPR) * V;
            if (c < C) r[i].get(p + c, C - c);
            else r[i].zero();
        }
    }
    __device__ __forceinline__ void put(T* p, int C, int l) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + i * TPR) * V;
            if (c < C) r[i].template put<true>(p + c, C - c);
        }
    }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) r[i].v[j] = x;
    }
    // f(vector, element) for every value of the row that this thread holds (values past C are left out)
    template <typename F>
    __device__ __forceinline__ static void each(int C, int l, F f) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if ((l + i * TPR) * V + j < C) f(i, j);
    }
};

// The row's sums of a and b, to every thread of it.  `slot` alternates between two LDS places from call to call, so one
// barrier per call is enough.
template <int TPR>
__device__ __forceinline__ void nm_sum2(float& a, float& b, float (*ws)[2][nm_waves(TPR)], int slot) {
#pragma unroll
    for (int d = 1; d < (TPR < MH_WAVE ? TPR : MH_WAVE); d <<= 1) {
        a += __shfl_xor(a, d, MH_WAVE);
        b += __shfl_xor(b, d, MH_WAVE);
    }
    if constexpr (TPR > MH_WAVE) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            ws[slot][0][w] = a;
            ws[slot][1][w] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int k = 0; k < TPR / MH_WAVE; ++k) {
            a += ws[slot][0][k];
            b += ws[slot][1][k];
        }
    }
}

// mean and 1 / sqrt(var + eps) of a row held in registers; the variance from the differences to the mean
template <int TY, int TPR, int NV, bool LAYER>
__device__ __forceinline__ void nm_stats(const nm_row<TY, TPR, NV>& y, int C, int l, float eps, float (*ws)[2][nm_waves(TPR)],
                                         int& slot, float& mean, float& rstd) {
    typedef nm_row<TY, TPR, NV> row;
    float s = 0.f, z = 0.f;
    mean = 0.f;
    if (LAYER) {
        row::each(C, l, [&](int i, int j) { s += y.r[i].v[j]; });
        nm_sum2<TPR>(s, z, ws, slot);
        slot ^= 1;
        mean = s / C;
        s = 0.f;
    }
    row::each(C, l, [&](int i, int j) {
        const float d = y.r[i].v[j] - mean;
        s += d * d;
    });
    nm_sum2<TPR>(s, z, ws, slot);
    slot ^= 1;
    rstd = 1.f / sqrtf(s / C + eps);
}

// GATE 0: none, 1: one value a row, 2: one a channel; Y: a branch y to add.  stats [T, 4]: mean and 1 / std of y and of h.
// Bound by its bytes: 32,768 rows of 2,048 bfloat16 channels with a gate each in 129 us (5.2 TB/s), 160 rows of 512 in 4.2 us.
template <int TY, int TPR, int NV, bool LAYER, bool Y, int GATE>
__device__ __forceinline__ void nm_fwd_body(const void* x_, const void* y_, const void* gate_, const void* scale_,
                                            const void* wp_, const void* wn_, void* h_, void* n_, float* stats, int T, int C,
                                            float eps) {
    typedef nm_row<TY, TPR, NV> row;
    typedef typename mm_type<TY>::t S;
    __shared__ float ws[2][2][nm_waves(TPR)];
    constexpr int PER = nm_rows(TPR);                     // rows of a workgroup
    const int l = threadIdx.x % TPR;
    const long long t = (long long)blockIdx.x * PER + threadIdx.x / TPR;
    if (t >= T) return;                                  // all threads of a row
    int slot = 0;
    row h, w;
    float my = 0.f, ry = 0.f, mh, rh;
    h.get(static_cast<const S*>(x_) + t * C, C, l);
    if (Y) {
        row y, k;
        y.get(static_cast<const S*>(y_) + t * C, C, l);
        if (GATE == 2) k.get(static_cast<const S*>(gate_) + t * C, C, l);
        nm_stats<TY, TPR, NV, LAYER>(y, C, l, eps, ws, slot, my, ry);
        const float gr = GATE == 1 ? mm_get<TY>(static_cast<const S*>(gate_) + t) : 1.f;
        row::each(C, l, [&](int i, int j) { y.r[i].v[j] = (y.r[i].v[j] - my) * ry; });
        if (wp_) {
            w.get(static_cast<const S*>(wp_), C, l);
            row::each(C, l, [&](int i, int j) { y.r[i].v[j] *= w.r[i].v[j]; });
        }
        if (scale_) {
            w.get(static_cast<const S*>(scale_), C, l);
            row::each(C, l, [&](int i, int j) { y.r[i].v[j] *= w.r[i].v[j]; });
        }
        row::each(C, l, [&](int i, int j) {
            h.r[i].v[j] += (GATE == 2 ? k.r[i].v[j] : GATE == 1 ? gr : 1.f) * y.r[i].v[j];
        });
        h.put(static_cast<S*>(h_) + t * C, C, l);
    }
    nm_stats<TY, TPR, NV, LAYER>(h, C, l, eps, ws, slot, mh, rh);
    if (wn_) w.get(static_cast<const S*>(wn_), C, l);
    else w.fill(1.f);
    row::each(C, l, [&](int i, int j) { h.r[i].v[j] = (h.r[i].v[j] - mh) * rh * w.r[i].v[j]; });
    h.put(static_cast<S*>(n_) + t * C, C, l);
    if (stats && l == 0) *reinterpret_cast<mh_f4*>(stats + 4 * t) = mh_f4{my, ry, mh, rh};
}

// The vectors of a row as they lie in memory: a quarter or half of their values' registers, so the next row's can be under
// way during this one's sums.
template <int TY, int TPR, int NV>
struct nm_raw {
    mh_u4 w[NV];
    __device__ __forceinline__ void get(const typename mm_type<TY>::t* p, int C, int l) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + i * TPR) * mm_vec<TY>::V;
            w[i] = c < C ? mm_vec<TY>::raw(p + c, C - c) : mh_u4{0u, 0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ nm_row<TY, TPR, NV> row() const {
        nm_row<TY, TPR, NV> r;
#pragma unroll
        for (int i = 0; i < NV; ++i) r.r[i].set(w[i]);
        return r;
    }
};

// Rows walked by a fixed number of row groups (a wave or a workgroup each).  With z = sum_t dh gate u, ds = wp z and dwp = s z:
// two sums over rows stay in registers and go to part[workgroup][3][C] (scale, wp, wn) at the end, added by mm_sum in order.
// Bound by its bytes, if the next row is loaded during this row's sums over the channels and the weights stay in registers:
// 32,768 rows of 2,048 bfloat16 channels with a gate each took 433 us without, 208 with it (5.2 TB/s, a large copy's rate).
template <int TY, int TPR, int NV, bool LAYER, bool Y, int GATE>
__device__ __forceinline__ void nm_bwd_body(const void* gh_, const void* gn_, const void* x_, const void* y_, const void* gate_,
                                            const void* scale_, const void* wp_, const void* wn_, const float* stats, void* dx_,
                                            void* dy_, void* dgate_, float* part, int T, int C) {
    typedef nm_row<TY, TPR, NV> row;
    typedef nm_raw<TY, TPR, NV> raw;
    typedef typename mm_type<TY>::t S;
    __shared__ float ws[2][2][nm_waves(TPR)];
    constexpr int PER = nm_rows(TPR);                     // rows of a workgroup
    const int l = threadIdx.x % TPR, groups = gridDim.x * PER;
    const int me = blockIdx.x * PER + threadIdx.x / TPR;
    int slot = 0;
    const S one = []() { if constexpr (TY == MM_F32) return 1.f; else return mm_round<TY>(1.f); }();
    raw rs, rp, rn;                                       // scale, wp, wn: ones where absent
    auto weight = [&](raw& r, const void* p) {
        if (p) r.get(static_cast<const S*>(p), C, l);
        else
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                unsigned w;
                if constexpr (TY == MM_F32) w = __float_as_uint(one);
                else w = one | (unsigned)one << 16;
                r.w[i] = mh_u4{w, w, w, w};
            }
    };
    if (Y) {
        weight(rs, scale_);
        weight(rp, wp_);
    }
    weight(rn, wn_);
    row az, an;
    az.fill(0.f);
    an.fill(0.f);
    struct inputs {
        raw x, y, gh, gn, k;
        float gr;
        mh_f4 st;
    } nx;
    auto load = [&](inputs& a, long long t) {
        a.st = *reinterpret_cast<const mh_f4*>(stats + 4 * t);
        a.x.get(static_cast<const S*>(x_) + t * C, C, l);
        if (Y) a.y.get(static_cast<const S*>(y_) + t * C, C, l);
        if (Y && GATE == 2) a.k.get(static_cast<const S*>(gate_) + t * C, C, l);
        if (Y && GATE == 1) a.gr = mm_get<TY>(static_cast<const S*>(gate_) + t);
        if (gn_) a.gn.get(static_cast<const S*>(gn_) + t * C, C, l);
        if (gh_) a.gh.get(static_cast<const S*>(gh_) + t * C, C, l);
    };
    if (me < T) load(nx, me);
    for (long long t = me; t < T; t += groups) {
        const mh_f4 st = nx.st;
        const float gr = Y && GATE == 1 ? nx.gr : 1.f;
        row v = nx.x.row(), u, q, w, k;
        if (Y) u = nx.y.row();
        if (Y && GATE == 2) k = nx.k.row();
        if (gn_) q = nx.gn.row();
        else q.fill(0.f);
        if (gh_) w = nx.gh.row();
        else w.fill(0.f);
        if (t + groups < T) load(nx, t + groups);
        if (Y) {
            const row s = rs.row(), p = rp.row();
            row::each(C, l, [&](int i, int j) {
                u.r[i].v[j] = (u.r[i].v[j] - st[0]) * st[1];
                v.r[i].v[j] += (GATE == 2 ? k.r[i].v[j] : gr) * s.r[i].v[j] * p.r[i].v[j] * u.r[i].v[j];
            });
        }
        float sv = 0.f, s1 = 0.f;
        {
            const row n = rn.row();
            row::each(C, l, [&](int i, int j) {
                const float h = (v.r[i].v[j] - st[2]) * st[3], g = q.r[i].v[j] * n.r[i].v[j];
                an.r[i].v[j] += q.r[i].v[j] * h;
                v.r[i].v[j] = h;
                q.r[i].v[j] = g;
                sv += g * h;
                if (LAYER) s1 += g;
            });
        }
        nm_sum2<TPR>(sv, s1, ws, slot);
        slot ^= 1;
        sv /= C;
        s1 /= C;
        row::each(C, l, [&](int i, int j) {              // w: dh
            w.r[i].v[j] += st[3] * (q.r[i].v[j] - v.r[i].v[j] * sv - s1);
        });
        if (dx_) w.put(static_cast<S*>(dx_) + t * C, C, l);
        if (Y) {
            const row s = rs.row(), p = rp.row();
            float se = 0.f, s0 = 0.f, sg = 0.f, z = 0.f;
            row::each(C, l, [&](int i, int j) {
                const float dh = w.r[i].v[j], g = GATE == 2 ? k.r[i].v[j] : gr, uu = u.r[i].v[j];
                const float sp = s.r[i].v[j] * p.r[i].v[j], dg = dh * uu * sp, e = dh * g * sp;
                az.r[i].v[j] += dh * g * uu;
                if (GATE == 1) sg += dg;
                if (GATE == 2) q.r[i].v[j] = dg;
                w.r[i].v[j] = e;
                se += e * uu;
                if (LAYER) s0 += e;
            });
            nm_sum2<TPR>(se, s0, ws, slot);
            slot ^= 1;
            se /= C;
            s0 /= C;
            row::each(C, l, [&](int i, int j) { w.r[i].v[j] = st[1] * (w.r[i].v[j] - u.r[i].v[j] * se - s0); });
            if (dy_) w.put(static_cast<S*>(dy_) + t * C, C, l);
            if (GATE == 2 && dgate_) q.put(static_cast<S*>(dgate_) + t * C, C, l);
            if (GATE == 1 && dgate_) {
                nm_sum2<TPR>(sg, z, ws, slot);
                slot ^= 1;
                if (l == 0) {
                    if constexpr (TY == MM_F32) static_cast<float*>(dgate_)[t] = sg;
                    else static_cast<unsigned short*>(dgate_)[t] = mm_round<TY>(sg);
                }
            }
        }
    }
    if (!part) return;
    float* p = part + (long long)blockIdx.x * 3 * C;
    if constexpr (PER > 1) {
        // a workgroup's rows add up in LDS, in their order
        __shared__ float sums[2][PER][TPR * NV * row::V];
        const int g = threadIdx.x / TPR;
        row::each(C, l, [&](int i, int j) {
            const int c = (l + i * TPR) * row::V + j;
            sums[0][g][c] = az.r[i].v[j];
            sums[1][g][c] = an.r[i].v[j];
        });
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += 256) {
            float z = sums[0][0][c], v = sums[1][0][c];
#pragma unroll 4
            for (int k = 1; k < PER; ++k) {
                z += sums[0][k][c];
                v += sums[1][k][c];
            }
            if (Y) {
                p[c] = wp_ ? z * mm_get<TY>(static_cast<const S*>(wp_) + c) : z;
                p[C + c] = scale_ ? z * mm_get<TY>(static_cast<const S*>(scale_) + c) : z;
            }
            p[2 * C + c] = v;
        }
        return;
    }
    row s, o;
    if (Y) {
        s = rs.row();
        o = rp.row();
    }
    row::each(C, l, [&](int i, int j) {
        const int c = (l + i * TPR) * row::V + j;
        if (Y) {
            p[c] = az.r[i].v[j] * o.r[i].v[j];
            p[C + c] = az.r[i].v[j] * s.r[i].v[j];
        }
        p[2 * C + c] = an.r[i].v[j];
    });
}
