// _layers.so — the trainable node layers (dense, expert_dense, dispatch, combine, block_norm) between torch and the C ABI.
//
// Each is an autograd function in C++ that allocates its results and calls the entry points of include/mace_hip.h on torch's
// current stream.  A call of a few microseconds of GPU work is its host work, most of all in a backward pass, which
// runs on a thread of the autograd engine that slept before.  Measured on layers of a few rows: 5.2 us forward (10.9 as Python
// functions over ctypes), 75 us forward and backward (125; of these the engine's own are 45).
//
// What depends on sizes, types and alignment alone (modules, tiles, pieces) is asked from Python once for each and kept
// (`plan`).  Arguments that do not fit come back as None, and the Python side, which knows the reasons, raises.  Handles in
// plans are of modules that Python keeps for the life of the process.
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <optional>
#include <unordered_map>

#include "../../include/mace_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
float* f32(const Tensor& t) { return static_cast<float*>(ptr(t)); }
int32_t* i32(const Tensor& t) { return static_cast<int32_t*>(ptr(t)); }
uint32_t* u32(const Tensor& t) { return static_cast<uint32_t*>(ptr(t)); }
uint16_t* u16(const Tensor& t) { return static_cast<uint16_t*>(ptr(t)); }
Tensor value(const Maybe& t) { return t.has_value() ? *t : Tensor(); }

void check(int rc, const char* what) {
    TORCH_CHECK(rc == 0, "mace_hip_kernels: ", what, " failed (code ", rc, "): ", mh_last_error());
}

// While launches are timed, Python's launch(tag, fn), which brackets fn() with events; else null.
std::atomic<PyObject*> g_timed{nullptr};

template <class F>
void launch(const char* tag, F f) {
    if (!g_timed.load(std::memory_order_relaxed)) return check(f(), tag);
    py::gil_scoped_acquire lock;
    if (PyObject* timed = g_timed.load()) {
        py::reinterpret_borrow<py::object>(timed)(tag, py::cpp_function([&f] { return f(); }));
    } else {
        check(f(), tag);
    }
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

// A saved tensor may have been given other data since (`p.data = ...`, a module moved to another device or type): the kernels
// would read that as what it was.
void unchanged(const Tensor& t, const Tensor& grad, at::ScalarType type, int64_t numel, int64_t last) {
    TORCH_CHECK(!t.defined() || (t.device() == grad.device() && t.scalar_type() == type && t.numel() == numel && t.dim() &&
                                 t.size(-1) == last),
                "mace_hip_kernels: a tensor of a trainable layer has changed its shape, type or device since its forward");
}

const char* const kDouble =
    "mace_hip_kernels: double backward (create_graph=True) is not available for the trainable node layers "
    "(dense, expert_dense, dispatch, combine, block_norm)";

// A tangent would be lost without a word where nothing asks for a gradient: the kernels then run without an autograd function.
void no_tangents(c10::ArrayRef<const Tensor*> inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                    "mace_hip_kernels: forward-mode derivatives are not available for the trainable node layers "
                                    "(dense, expert_dense, dispatch, combine, block_norm)");
}

// ---------------------------------------------------------------------------------------------------------- plans
enum { FORWARD, BACKWARD, ROUTE, NORM };
// a kind of plan and what it depends on, in the order of Python's planner of that kind
struct Key {
    std::array<int64_t, 13> v{};
    bool operator==(const Key& o) const { return v == o.v; }
};
struct KeyHash {
    size_t operator()(const Key& k) const {
        uint64_t h = 0;
        for (int64_t x : k.v) {
            h = (h ^ static_cast<uint64_t>(x)) * 0x9E3779B97F4A7C15ull;
            h ^= h >> 29;
        }
        return static_cast<size_t>(h);
    }
};

// the numbers that Python's planner gives for a key (their meaning: the enums below)
struct Plan : torch::CustomClassHolder {
    Key key;
    std::vector<int64_t> n;
    int64_t operator[](int i) const { return n[i]; }
    mh_module* module(int i) const { return reinterpret_cast<mh_module*>(n[i]); }
};
typedef c10::intrusive_ptr<Plan> PlanPtr;

PyObject* g_planner = nullptr;                          // both touched with the interpreter's lock held only
std::unordered_map<Key, PlanPtr, KeyHash> g_plans;

PlanPtr plan(const Key& key, size_t numbers) {
    auto it = g_plans.find(key);
    if (it != g_plans.end()) return it->second;
    TORCH_CHECK(g_planner, "mace_hip_kernels: the trainable layers have no planner");
    py::tuple args(key.v.size());
    for (size_t k = 0; k < key.v.size(); ++k) args[k] = key.v[k];
    PlanPtr p = c10::make_intrusive<Plan>();
    p->key = key;
    p->n = py::reinterpret_borrow<py::object>(g_planner)(*args).cast<std::vector<int64_t>>();
    TORCH_CHECK(p->n.size() == numbers, "mace_hip_kernels: the planner gave ", p->n.size(), " numbers, not ", numbers);
    if (g_plans.size() >= 65536) g_plans.clear();        // sizes that change with every call do not pile up
    g_plans.emplace(key, p);
    return p;
}

PlanPtr saved_plan(AutogradContext* ctx) {
    return c10::static_intrusive_pointer_cast<Plan>(ctx->saved_data["p"].toCapsule());
}

// rows [R, width] whose elements are contiguous (copied only where they are not), and the distance between them
Tensor rows_of(const Tensor& t, int64_t width, int64_t* ld) {
    Tensor r = t;
    if (t.dim() != 2) {
        int64_t rows = 1;
        for (int64_t k = 0; k + 1 < t.dim(); ++k) rows *= t.size(k);
        r = t.reshape({rows, width});
    }
    if (r.size(0) <= 1 || width == 0) {
        *ld = width;
        return r.contiguous();
    }
    if ((width > 1 && r.stride(1) != 1) || r.stride(0) < width) r = r.contiguous();
    *ld = r.stride(0);
    return r;
}

const int64_t kMost = (1LL << 31) - 1024;               // rows, and values of one
const int64_t kSteps = 1 << 21;                         // values between rows that a tile loads straight to LDS (its 31-bit offsets)

// whether rows of a 16-bit tensor are whole steps of 16 bytes, with a tile's offsets within 2^31 bytes
bool steps(const Tensor& t, int64_t ld, int64_t width) {
    return width % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && ld < kSteps;
}

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// ---------------------------------------------------------------------------------------------------------- dense
enum { F_MODULE, F_HALVES, F_SPLIT, F_SUMS, F_PAD_X, F_PAD_W, F_SIZE };
enum { B_SUMS, B_ROWS, B_OUTER, B_SPLIT, B_LS, B_SLOTS, B_LO, B_SLOTS_O, B_SCRATCH, B_DX_HALVES, B_DW_HALVES, B_PAD_G, B_PAD_W,
       B_PAD_X, B_SIZE };

Tensor padded(mh_module* sums, const Tensor& t, int64_t* ld, int64_t rows, int64_t width) {
    const int64_t to = up(width, 8);
    TORCH_CHECK(rows < kMost && to < kSteps, "mace_hip_kernels: rows that no tile takes were to be copied for one");
    Tensor y = at::empty({rows, to}, t.options());
    launch("mm_pad", [&] { return mh_mm_pad(sums, ptr(t), *ld, ptr(y), rows, width, to, stream_of(t)); });
    *ld = to;
    return y;
}

struct Halves {
    Tensor y, peak;
};

Halves halves_of_rows(mh_module* split, const Tensor& x, int64_t ld, int64_t R, int64_t K) {
    Halves h{at::empty({R * 2 * up(K, 32)}, x.options().dtype(at::kUInt16)), at::empty({R + 1}, x.options().dtype(at::kInt))};
    launch("hv_rows", [&] { return mh_hv_rows(split, f32(x), ld, u16(h.y), u32(h.peak), R, K, stream_of(x)); });
    return h;
}

// columns scaled per group of rows: by offsets, else equal groups; peak [2][groups][C] and a word more
Halves halves_of_columns(mh_module* split, const Tensor& x, int64_t ld, int64_t R, int64_t C, int64_t groups,
                         const Tensor& off) {
    Halves h{at::empty({R * 2 * up(C, 8)}, x.options().dtype(at::kUInt16)),
             at::zeros({2 * groups * C + 1}, x.options().dtype(at::kInt))};
    const int64_t G = off.defined() ? 0 : R / groups;
    // pieces of rows for about eight workgroups per compute unit
    const int64_t L = std::min<int64_t>(256, std::max<int64_t>(16, up((R * ((C + 255) / 256) + 2047) / 2048, 4)));
    const int64_t slots = off.defined() ? (R + L - 1) / L + groups : groups * ((G + L - 1) / L);
    launch("hv_columns", [&] {
        return mh_hv_columns(split, f32(x), ld, u16(h.y), u32(h.peak), i32(off), R, C, groups, G, L, slots, stream_of(x));
    });
    return h;
}

// workgroups that compute marked tiles again: three on each compute unit
const int kAgain = 768;

struct DenseArgs {
    Tensor x, w;         // x [R, K] with ld between rows, w contiguous
    int64_t ld, R, n, K, groups, act;
    bool x_ok, w_ok;     // of 16-bit types: whole steps
};

DenseArgs dense_args(const Tensor& x, const Tensor& w, bool grouped, int64_t act) {
    DenseArgs a;
    a.K = w.size(-1), a.n = w.size(-2), a.groups = grouped ? w.size(0) : 1, a.act = act;
    a.x = rows_of(x, a.K, &a.ld);
    a.w = w.contiguous();
    a.R = a.x.size(0);
    const bool f = x.scalar_type() == at::kFloat;
    a.x_ok = !f && steps(a.x, a.ld, a.K), a.w_ok = !f && steps(a.w, a.K, a.K);
    return a;
}

// act(x w^T + b) + res, and act' of it where `slope`
Tensor dense_forward(DenseArgs a, const Tensor& like, const Tensor& b, const Tensor& res, const Tensor& off, Tensor* slope) {
    const int64_t R = a.R, K = a.K, n = a.n, groups = a.groups;
    c10::SmallVector<int64_t, 5> shape(like.sizes().begin(), like.sizes().end());
    shape.back() = n;
    Tensor out = at::empty(shape, like.options());
    const bool f = like.scalar_type() == at::kFloat;
    if (slope) *slope = at::empty({R, n}, like.options().dtype(f ? at::kFloat : at::kUInt16));
    if (!R || !n) return out;
    const PlanPtr pp = plan(Key{{FORWARD, like.device().index(), type_of(like), R, n, K, groups, a.act, a.x_ok, a.w_ok}}, F_SIZE);
    const Plan& p = *pp;
    int64_t ldr = 0, ldw = std::max<int64_t>(1, K);
    const Tensor r = res.defined() ? rows_of(res, n, &ldr) : Tensor();
    void* s = stream_of(like);
    void* sl = slope ? ptr(*slope) : nullptr;
    if (p[F_HALVES]) {
        const Halves h = halves_of_rows(p.module(F_SPLIT), a.x, a.ld, R, K);
        const Halves c = halves_of_rows(p.module(F_SPLIT), a.w, K, groups * n, K);
        launch("hv_fwd", [&] {
            return mh_hv_mm(p.module(F_MODULE), u16(h.y), u16(c.y), f32(out), f32(b), f32(r), ldr, static_cast<float*>(sl),
                            i32(off), u32(h.peak), u32(c.peak), nullptr, R, n, K, groups, s);
        });
        launch("hv_again", [&] {
            return mh_hv_again_mm(p.module(F_MODULE), f32(a.x), a.ld, f32(a.w), K, f32(out), f32(b), f32(r), ldr,
                                  static_cast<float*>(sl), i32(off), u32(h.peak), u32(c.peak), nullptr, R, n, K, groups, kAgain, s);
        });
        return out;
    }
    if (p[F_PAD_X]) a.x = padded(p.module(F_SUMS), a.x, &a.ld, R, K);
    if (p[F_PAD_W]) a.w = padded(p.module(F_SUMS), a.w, &ldw, groups * n, K);
    launch("mm_fwd", [&] {
        return mh_mm_rows(p.module(F_MODULE), ptr(a.x), a.ld, ptr(a.w), ldw, ptr(out), ptr(b), ptr(r), ldr, sl, i32(off), R, n, K,
                          groups, s);
    });
    return out;
}

struct DenseFn : torch::autograd::Function<DenseFn> {
    // need: bits of x, w, b, res
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& res,
                          const Maybe& off, int64_t act, int64_t need) {
        const DenseArgs a = dense_args(x, w, off.has_value(), act);
        const bool made = act != 0 && (need & 7), f = x.scalar_type() == at::kFloat;
        Tensor slope;
        Tensor out = dense_forward(a, x, b ? b->contiguous() : Tensor(), value(res), value(off), made ? &slope : nullptr);
        ctx->save_for_backward({need & 2 ? x : Tensor(), need & 1 ? a.w : Tensor(), slope, value(off)});
        if (need & 7) {
            // g is taken to come in whole steps where it can; the backward asks again where it does not
            ctx->saved_data["p"] = c10::IValue::make_capsule(plan(
                Key{{BACKWARD, x.device().index(), type_of(x), a.R, a.n, a.K, a.groups, off.has_value(), made,
                     made || f || a.n % 8 == 0, (need & 1) && a.w_ok, (need & 2) && a.x_ok, need & 7}}, B_SIZE));
            ctx->saved_data["x"] = x.sizes().vec();
        }
        ctx->saved_data["n"] = need;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), kDouble);
        variable_list out(7);
        const int64_t need = ctx->saved_data["n"].toInt();
        if (need & 8) out[3] = grads[0];
        if (!(need & 7)) return out;
        const auto saved = ctx->get_saved_variables();
        PlanPtr pp = saved_plan(ctx);
        Key key = pp->key;
        const int64_t R = key.v[3], N = key.v[4], K = key.v[5], groups = key.v[6];
        const bool grouped = key.v[7], made = key.v[8];
        Tensor x = saved[0], w = saved[1];
        const Tensor &slope = saved[2], &off = saved[3];
        int64_t ldg, ldx = 0, ldw = std::max<int64_t>(1, K), ldp = 0;
        Tensor g = rows_of(grads[0], N, &ldg);
        const bool f = g.scalar_type() == at::kFloat;
        unchanged(x, g, g.scalar_type(), R * K, K);
        unchanged(w, g, g.scalar_type(), groups * N * K, K);
        unchanged(off, g, at::kInt, groups + 1, groups + 1);
        if (x.defined()) x = rows_of(x, K, &ldx);
        if (w.defined()) w = w.contiguous();
        key.v[9] = made || f || steps(g, ldg, N);
        key.v[10] = w.defined() && !f && steps(w, K, K);
        key.v[11] = x.defined() && !f && steps(x, ldx, K);
        if (!(key == pp->key)) {
            py::gil_scoped_acquire lock;
            pp = plan(key, B_SIZE);
        }
        const Plan& p = *pp;
        mh_module* sums = p.module(B_SUMS);
        Tensor prod;
        if (made) {
            ldp = f ? N : up(N, 8);
            prod = at::empty({R, ldp}, g.options());
        } else if (p[B_PAD_G]) {
            g = padded(sums, g, &ldg, R, N);
        }
        if (p[B_PAD_W]) w = padded(sums, w, &ldw, groups * N, K);
        if (p[B_PAD_X]) x = padded(sums, x, &ldx, R, K);
        Tensor dx, dw, db, part;
        const auto of = [&](std::initializer_list<int64_t> shape) {
            return at::empty(at::IntArrayRef(shape.begin() + !grouped, shape.end()), g.options());
        };
        if (need & 1) dx = at::empty(ctx->saved_data["x"].toDimVector(), g.options());
        if (need & 2) dw = of({groups, N, K});
        if (need & 4) db = of({groups, N});
        if (p[B_SCRATCH]) part = at::empty({p[B_SCRATCH]}, g.options().dtype(at::kFloat));
        void* s = stream_of(g);
        mh_module* rows = p[B_DX_HALVES] ? nullptr : p.module(B_ROWS);
        mh_module* outer = p[B_DW_HALVES] ? nullptr : p.module(B_OUTER);
        if (made || (need & 4) || rows || outer)
            launch("mm_bwd", [&] {
                return mh_mm_bwd(sums, rows, outer, ptr(g), ldg, ptr(slope), ptr(w), ldw, ptr(x), ldx, i32(off), ptr(prod), ldp,
                                 rows ? ptr(dx) : nullptr, outer ? ptr(dw) : nullptr, ptr(db), f32(part), R, N, K, groups,
                                 p[B_LS], p[B_SLOTS], p[B_LO], p[B_SLOTS_O], s);
            });
        if (made) {
            g = prod;
            ldg = ldp;
        }
        mh_module* split = p.module(B_SPLIT);
        if (p[B_DX_HALVES]) {
            const Halves a = halves_of_rows(split, g, ldg, R, N);
            const Halves c = halves_of_columns(split, w, K, groups * N, K, groups, Tensor());
            launch("hv_dx", [&] {
                return mh_hv_mm(p.module(B_ROWS), u16(a.y), u16(c.y), f32(dx), nullptr, nullptr, 0, nullptr, i32(off),
                                u32(a.peak), u32(c.peak), u32(c.peak) + groups * K, R, K, N, groups, s);
            });
            launch("hv_again", [&] {
                return mh_hv_again_mm(p.module(B_ROWS), f32(g), ldg, f32(w), K, f32(dx), nullptr, nullptr, 0, nullptr, i32(off),
                                      u32(a.peak), u32(c.peak), u32(c.peak) + groups * K, R, K, N, groups, kAgain, s);
            });
        }
        if (p[B_DW_HALVES]) {
            const Halves a = halves_of_columns(split, g, ldg, R, N, groups, off);
            const Halves c = halves_of_columns(split, x, ldx, R, K, groups, off);
            launch("hv_dw", [&] {
                return mh_hv_outer(p.module(B_OUTER), u16(a.y), u16(c.y), f32(dw), f32(part), i32(off), u32(a.peak),
                                   u32(a.peak) + groups * N, u32(c.peak), u32(c.peak) + groups * K, R, N, K, groups, p[B_LO],
                                   p[B_SLOTS_O], s);
            });
            launch("hv_again", [&] {
                return mh_hv_again_outer(p.module(B_OUTER), f32(g), ldg, f32(x), ldx, f32(dw), f32(part), i32(off), u32(a.peak),
                                         u32(a.peak) + groups * N, u32(c.peak), u32(c.peak) + groups * K, R, N, K, groups,
                                         p[B_LO], p[B_SLOTS_O], kAgain, s);
            });
            if (p[B_LO])
                launch("mm_sum", [&] { return mh_mm_sum(sums, f32(part), ptr(dw), i32(off), R, groups, p[B_LO], N * K, s); });
        }
        out[0] = dx;
        out[1] = dw;
        out[2] = db;
        return out;
    }
};

bool tensor(py::handle h, Tensor* t) {
    if (!THPVariable_Check(h.ptr())) return false;
    *t = THPVariable_Unpack(h.ptr());
    return true;
}
bool maybe(py::handle h, Tensor* t) { return h.is_none() || tensor(h, t); }
bool alike(const Tensor& t, const Tensor& x) { return t.scalar_type() == x.scalar_type() && t.device() == x.device(); }
// rows of features that the kernels take
bool fits(const Tensor& x) {
    return x.is_cuda() && type_of(x) >= 0 && x.dim() >= 1 && x.size(-1) < kMost &&
           x.numel() / std::max<int64_t>(1, x.size(-1)) < kMost;
}
bool like_rows(const Tensor& t, const Tensor& x, int64_t width) {
    if (!alike(t, x) || t.dim() != x.dim() || t.size(-1) != width) return false;
    for (int64_t k = 0; k + 1 < x.dim(); ++k)
        if (t.size(k) != x.size(k)) return false;
    return true;
}
Maybe opt(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
bool grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// dense (offsets None) and expert_dense; None where an argument does not fit
py::object dense(py::handle x_, py::handle w_, py::handle b_, py::handle r_, int64_t act, py::handle o_) {
    Tensor x, w, b, r, off;
    if (!tensor(x_, &x) || !tensor(w_, &w) || !maybe(b_, &b) || !maybe(r_, &r) || !maybe(o_, &off) || act < 0 || !fits(x) ||
        !alike(w, x))
        return py::none();
    const bool grouped = off.defined();
    if (w.dim() != (grouped ? 3 : 2) || w.size(-1) != x.size(-1)) return py::none();
    const int64_t n = w.size(-2), groups = grouped ? w.size(0) : 1;
    if (b.defined() && (!alike(b, x) || b.dim() != w.dim() - 1 || b.size(-1) != n || (grouped && b.size(0) != groups)))
        return py::none();
    if (r.defined() && !like_rows(r, x, n)) return py::none();
    if (grouped && (x.dim() != 2 || groups < 1 || off.scalar_type() != at::kInt || off.device() != x.device() ||
                    off.dim() != 1 || off.size(0) != groups + 1))
        return py::none();
    no_tangents({&x, &w, &b, &r});
    if (grouped) off = off.contiguous();
    int64_t need = 0;
    if (at::GradMode::is_enabled()) need = grad(x) | grad(w) << 1 | grad(b) << 2 | grad(r) << 3;
    if (need) return py::cast(DenseFn::apply(x, w, opt(b), opt(r), opt(off), act, need));
    return py::cast(dense_forward(dense_args(x, w, grouped, act), x, b.defined() ? b.contiguous() : b, r, off, nullptr));
}

// ---------------------------------------------------------------------------------------------------------- routing
enum { R_MODULE, R_LANES, R_SIZE };                     // the sort for no type (-1), else the rows of a type

PlanPtr route_plan(const Tensor& t, int64_t C) {
    return plan(Key{{ROUTE, t.device().index(), type_of(t), C}}, R_SIZE);
}

// a tensor of its own on part of `buf`'s memory (a view by the dispatcher costs 0.8 us, of a call of 6)
Tensor part_of(const Tensor& buf, int64_t first, c10::IntArrayRef shape) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(first);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    return t;
}

py::object expert_order(py::handle e_, int64_t E) {
    Tensor e;
    if (!tensor(e_, &e) || !e.is_cuda() || (e.scalar_type() != at::kInt && e.scalar_type() != at::kLong) || e.dim() != 2 ||
        e.size(1) < 1 || E < 1 || E > 1024 || e.numel() >= (1LL << 31) - (1 << 21))
        return py::none();
    e = e.contiguous();
    const int64_t A = e.numel();
    const PlanPtr p = plan(Key{{ROUTE, e.device().index(), -1, 0}}, R_SIZE);
    // workgroups of 4,096 assignments, 512 at most
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(512, (A + 4095) / 4096));
    Tensor buf = at::empty({E + 1 + 2 * A + (blocks > 1 ? blocks * (E + 1) : 0)}, e.options().dtype(at::kInt));
    int32_t* d = i32(buf);
    launch("expert_order", [&] {
        return mh_expert_order(p->module(R_MODULE), ptr(e), e.scalar_type() == at::kLong, A, E,
                               blocks > 1 ? d + E + 1 + 2 * A : nullptr, blocks, d, d + E + 1, d + E + 1 + A, stream_of(e));
    });
    return py::make_tuple(part_of(buf, 0, {E + 1}), part_of(buf, E + 1, {A}), part_of(buf, E + 1 + A, e.sizes()));
}

// x [T, C] to its places [T k, C]
Tensor spread(const Plan& p, const Tensor& x, const Tensor& place, const Tensor& off) {
    const int64_t T = place.size(0), k = place.size(1), C = x.size(1);
    Tensor y = at::empty({T * k, C}, x.options());
    if (!T || !C) return y;
    int64_t ld;
    const Tensor x2 = rows_of(x, C, &ld);
    launch("ex_dispatch", [&] {
        return mh_dispatch(p.module(R_MODULE), ptr(x2), ld, i32(place), i32(off), ptr(y), T, k, C, off.size(0) - 1, p[R_LANES],
                           stream_of(x));
    });
    return y;
}

// res + sum_j w y[place] [T, C]
Tensor gather(const Plan& p, const Tensor& y, const Tensor& w, const Tensor& place, const Tensor& res) {
    const int64_t T = place.size(0), k = place.size(1), C = y.size(1);
    Tensor out = at::empty({T, C}, y.options());
    if (!T || !C) return out;
    int64_t ldr = 0;
    const Tensor y2 = y.contiguous(), r = res.defined() ? rows_of(res, C, &ldr) : Tensor();
    launch("ex_combine", [&] {
        return mh_combine(p.module(R_MODULE), ptr(y2), f32(w), i32(place), ptr(r), ldr, ptr(out), T, k, C, p[R_LANES],
                          stream_of(y));
    });
    return out;
}

struct DispatchFn : torch::autograd::Function<DispatchFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& place, const Tensor& off, const PlanPtr& p) {
        ctx->save_for_backward({place});
        ctx->saved_data["p"] = c10::IValue::make_capsule(p);
        return spread(*p, x, place, off);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), kDouble);
        const PlanPtr p = saved_plan(ctx);
        variable_list out(4);
        out[0] = gather(*p, grads[0], Tensor(), ctx->get_saved_variables()[0], Tensor());
        return out;
    }
};

struct CombineFn : torch::autograd::Function<CombineFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y, const Maybe& w, const Maybe& res, const Tensor& place,
                          const Tensor& off, const PlanPtr& p, int64_t need) {
        const Tensor wc = w ? w->contiguous() : Tensor();
        ctx->save_for_backward({need & 2 ? y : Tensor(), wc, place, off});
        ctx->saved_data["p"] = c10::IValue::make_capsule(p);
        ctx->saved_data["n"] = need;
        return gather(*p, y, wc, place, value(res));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), kDouble);
        const auto saved = ctx->get_saved_variables();
        const PlanPtr p = saved_plan(ctx);
        const int64_t need = ctx->saved_data["n"].toInt();
        const Tensor &place = saved[2], &off = saved[3];
        const int64_t T = place.size(0), k = place.size(1), C = grads[0].size(1);
        variable_list out(7);
        if (need & 4) out[2] = grads[0];
        if (!(need & 3)) return out;
        int64_t ldg;
        if (need & 2) unchanged(saved[0], grads[0], grads[0].scalar_type(), T * k * C, C);
        unchanged(saved[1], grads[0], at::kFloat, T * k, k);
        const Tensor g = rows_of(grads[0], C, &ldg), y = need & 2 ? saved[0].contiguous() : Tensor();
        const Tensor w = saved[1].defined() ? saved[1].contiguous() : Tensor();
        if (need & 1) out[0] = at::empty({T * k, C}, g.options());
        if (need & 2) out[1] = at::empty({T, k}, g.options().dtype(at::kFloat));
        if (T && (C || (need & 2)))
            launch("ex_combine_bwd", [&] {
                return mh_combine_bwd(p->module(R_MODULE), ptr(g), ldg, ptr(y), f32(w), i32(place), i32(off), ptr(out[0]),
                                      f32(out[1]), T, k, C, off.size(0) - 1, (*p)[R_LANES], stream_of(g));
            });
        return out;
    }
};

// places [T, k] and offsets [E + 1] as expert_order makes them: what the kernels read as rows of int32
bool an_order(const Tensor& place, const Tensor& off, const Tensor& x) {
    return place.device() == x.device() && off.device() == x.device() && place.scalar_type() == at::kInt &&
           off.scalar_type() == at::kInt && place.dim() == 2 && off.dim() == 1 && place.size(1) >= 1 && off.size(0) >= 2 &&
           place.is_contiguous() && off.is_contiguous() && place.numel() < kMost;
}

py::object dispatch(py::handle x_, const Tensor& place, const Tensor& off) {
    Tensor x;
    if (!tensor(x_, &x) || !fits(x) || x.dim() != 2 || !an_order(place, off, x) || x.size(0) != place.size(0)) return py::none();
    no_tangents({&x});
    const PlanPtr p = route_plan(x, x.size(1));
    if (at::GradMode::is_enabled() && grad(x)) return py::cast(DispatchFn::apply(x, place, off, p));
    return py::cast(spread(*p, x, place, off));
}

py::object combine(py::handle y_, py::handle w_, py::handle r_, const Tensor& place, const Tensor& off) {
    Tensor y, w, r;
    if (!tensor(y_, &y) || !maybe(w_, &w) || !maybe(r_, &r) || !fits(y) || y.dim() != 2 || !an_order(place, off, y) ||
        y.size(0) != place.numel())
        return py::none();
    if (w.defined() && (w.scalar_type() != at::kFloat || w.device() != y.device() || w.sizes() != place.sizes())) return py::none();
    if (r.defined() && (!alike(r, y) || r.dim() != 2 || r.size(0) != place.size(0) || r.size(1) != y.size(1))) return py::none();
    no_tangents({&y, &w, &r});
    const PlanPtr p = route_plan(y, y.size(1));
    int64_t need = 0;
    if (at::GradMode::is_enabled()) need = grad(y) | grad(w) << 1 | grad(r) << 2;
    if (need) return py::cast(CombineFn::apply(y, opt(w), opt(r), place, off, p, need));
    return py::cast(gather(*p, y, w.defined() ? w.contiguous() : w, place, r));
}

// ---------------------------------------------------------------------------------------------------------- norms
enum { N_MODULE, N_SUMS, N_BLOCKS, N_SIZE };

struct NormOut {
    Tensor h, n, stats;
};

NormOut norm_forward(const Plan& p, const Tensor& x, const Tensor& y, const Tensor& gate, const Tensor& scale, const Tensor& wp,
                     const Tensor& wn, double eps, bool keep) {
    const int64_t C = x.size(-1), T = x.numel() / C;
    NormOut o{y.defined() ? at::empty(x.sizes(), x.options()) : x, at::empty(x.sizes(), x.options()), Tensor()};
    if (keep) o.stats = at::empty({T, 4}, x.options().dtype(at::kFloat));
    if (T)
        launch("nm_fwd", [&] {
            return mh_norm_fwd(p.module(N_MODULE), ptr(x), ptr(y), ptr(gate), ptr(scale), ptr(wp), ptr(wn),
                               y.defined() ? ptr(o.h) : nullptr, ptr(o.n), f32(o.stats), T, C, static_cast<float>(eps),
                               stream_of(x));
        });
    return o;
}

struct NormFn : torch::autograd::Function<NormFn> {
    // need: bits of x, y, gate, scale, wp, wn
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& scale,
                                 const Maybe& wp, const Maybe& wn, double eps, const PlanPtr& p, int64_t need) {
        NormOut o = norm_forward(*p, x, value(y), value(gate), value(scale), value(wp), value(wn), eps, true);
        ctx->save_for_backward({x, value(y), value(gate), value(scale), value(wp), value(wn), o.stats});
        ctx->saved_data["p"] = c10::IValue::make_capsule(p);
        ctx->saved_data["n"] = need;
        ctx->set_materialize_grads(false);
        if (y) return {o.h, o.n};
        return {o.n};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), kDouble);
        auto s = ctx->get_saved_variables();
        const PlanPtr p = saved_plan(ctx);
        const int64_t need = ctx->saved_data["n"].toInt();
        const Tensor &x = s[0], &y = s[1], &gate = s[2];
        variable_list out(9);
        Tensor gh = y.defined() ? grads[0] : Tensor(), gn = grads.back();
        if (!gh.defined() && !gn.defined()) return out;
        if (gh.defined()) gh = gh.contiguous();
        if (gn.defined()) gn = gn.contiguous();
        const int64_t T = p->key.v[3], C = p->key.v[4];
        const int64_t gates = p->key.v[7] == 1 ? 1 : C, numel[6] = {T * C, T * C, T * gates, C, C, C};
        for (int k = 0; k < 6; ++k) {
            if (!s[k].defined()) continue;
            unchanged(s[k], gn.defined() ? gn : gh, (gn.defined() ? gn : gh).scalar_type(), numel[k], k == 2 ? gates : C);
            s[k] = s[k].contiguous();
        }
        if (need & 1) out[0] = at::empty(x.sizes(), x.options());
        if (need & 2) out[1] = at::empty(x.sizes(), x.options());
        if (need & 4) out[2] = at::empty(gate.sizes(), x.options());
        Tensor dw, part;
        const int64_t blocks = (*p)[N_BLOCKS];
        if (need >> 3) {
            dw = at::empty({3, C}, x.options());
            part = at::empty({blocks, 3, C}, x.options().dtype(at::kFloat));
        }
        launch("nm_bwd", [&] {
            return mh_norm_bwd(p->module(N_MODULE), p->module(N_SUMS), ptr(gh), ptr(gn), ptr(x), ptr(y), ptr(gate), ptr(s[3]),
                               ptr(s[4]), ptr(s[5]), f32(s[6]), ptr(out[0]), ptr(out[1]), ptr(out[2]), f32(part), ptr(dw), T, C,
                               blocks, stream_of(x));
        });
        for (int k = 0; k < 3; ++k)
            if (need >> (3 + k) & 1) out[3 + k] = dw.select(0, k);
        return out;
    }
};

py::object block_norm(py::handle x_, py::handle y_, py::handle g_, py::handle s_, py::handle wp_, py::handle wn_, double eps,
                      int64_t layer) {
    Tensor x, y, gate, scale, wp, wn;
    if (!tensor(x_, &x) || !maybe(y_, &y) || !maybe(g_, &gate) || !maybe(s_, &scale) || !maybe(wp_, &wp) || !maybe(wn_, &wn) ||
        !fits(x) || layer < 0 || !(eps >= 0))
        return py::none();
    const int64_t C = x.size(-1);
    if (C < 1 || C > 8192) return py::none();
    if (!y.defined() ? gate.defined() || scale.defined() || wp.defined() : !like_rows(y, x, C)) return py::none();
    int64_t mode = 0;
    if (gate.defined()) {
        const int64_t width = gate.dim() ? gate.size(-1) : 0;
        if ((width != 1 && width != C) || !like_rows(gate, x, width)) return py::none();
        mode = width == 1 ? 1 : 2;                       // one value a row, also where there is one channel
    }
    for (Tensor* t : {&scale, &wp, &wn}) {
        if (!t->defined()) continue;
        if (!alike(*t, x) || t->dim() != 1 || t->size(0) != C) return py::none();
    }
    no_tangents({&x, &y, &gate, &scale, &wp, &wn});
    for (Tensor* t : {&x, &y, &gate, &scale, &wp, &wn})
        if (t->defined()) *t = t->contiguous();
    const PlanPtr p = plan(Key{{NORM, x.device().index(), type_of(x), x.numel() / C, C, layer, y.defined(), mode}}, N_SIZE);
    int64_t need = 0;
    if (at::GradMode::is_enabled())
        need = grad(x) | grad(y) << 1 | grad(gate) << 2 | grad(scale) << 3 | grad(wp) << 4 | grad(wn) << 5;
    if (!need) {
        const NormOut o = norm_forward(*p, x, y, gate, scale, wp, wn, eps, false);
        return y.defined() ? py::make_tuple(o.h, o.n) : py::make_tuple(py::reinterpret_borrow<py::object>(x_), o.n);
    }
    const variable_list o = NormFn::apply(x, opt(y), opt(gate), opt(scale), opt(wp), opt(wn), eps, p, need);
    return y.defined() ? py::make_tuple(o[0], o[1]) : py::make_tuple(py::reinterpret_borrow<py::object>(x_), o[0]);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.attr("abi") = MH_ABI_VERSION;                      // of the header that this was built with
    // planner(kind, ...) -> numbers; timed: launch(tag, fn) while launches are timed, else None
    m.def("set_planner", [](py::object f) { g_planner = f.release().ptr(); });
    m.def("set_timed", [](py::object f) { Py_XDECREF(g_timed.exchange(f.is_none() ? nullptr : f.release().ptr())); });
    m.def("clear_plans", [] { g_plans.clear(); });
    m.def("dense", &dense);
    m.def("expert_order", &expert_order);
    m.def("dispatch", &dispatch);
    m.def("combine", &combine);
    m.def("block_norm", &block_norm);
}
