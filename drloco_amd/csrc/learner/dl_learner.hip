// dl_learner.hip -- extern "C" API of include/drloco_learner.h: argument checks, the choice of a kernel's form, launches.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <cmath>
#include <string>

#include "drloco_learner.h"
#include "dl_memory.hpp"
#include "dl_orth.hpp"

namespace {

thread_local std::string g_err;
int fail(int code, const char* what) noexcept {
    try { g_err = what; } catch (...) {}
    return code;
}
int launched(const char* what) noexcept {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return DL_OK;
    try { g_err = std::string(what) + ": " + hipGetErrorString(e); } catch (...) {}
    return DL_E_HIP;
}
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p % (uintptr_t)bytes) == 0; }
int elem_bytes(int dtype) { return dtype == DL_F32 ? 4 : 2; }

bool fits(int64_t blocks, int64_t threads) { return blocks <= 0xffffffff / threads; }          // a launch has less than 2^32 threads

// ---- gated memory ----
constexpr int64_t MAX_DIM = (int64_t)1 << 40;

const char* memory_shape_error(const dl_memory_shape* s) {
    if (!s) return "shape must not be NULL";
    if (s->dtype != DL_F32 && s->dtype != DL_BF16 && s->dtype != DL_F16) return "unknown dtype";
    if (s->reserved != 0) return "reserved must be 0";
    if (s->T < 0 || s->N < 0 || s->D < 0 || s->T > MAX_DIM || s->N > MAX_DIM || s->D > MAX_DIM) return "T, N and D must not be negative (nor above 2^40)";
    if (s->T > (1 << 30)) return "more than 2^30 steps";
    if ((__int128)s->T * s->N * s->D > ((__int128)1 << 46)) return "more than 2^46 elements";
    for (int64_t st : {s->x_t, s->x_n, s->gate_t, s->gate_n, s->starts_t, s->starts_n, s->grad_t, s->grad_n})
        if (st < 0) return "negative strides";
    // 64 walkers' rows are addressed with 32 bits
    const int64_t walkers = std::min<int64_t>(s->N, s->D ? 256 / s->D + 2 : 1), far = (int64_t)1 << 29;
    if (s->D > far) return "more than 2^29 channels";
    if (walkers > 1 && (s->x_n >= far / walkers || s->gate_n >= far / walkers || s->grad_n >= far / walkers || s->D >= far / walkers)) return "walkers too far apart (2^29 elements over the 64 lanes of a wave): pass a time-major copy";
    return nullptr;
}

// The form of a launch (dl_memory.hpp): V columns per lane, `blocks` waves across the columns, W waves of a workgroup along time and
// `chunks` such workgroups in a chain.
struct form { int V, W; int64_t chunks, blocks; };

// Columns per lane: eight bytes forward, four backward, where three arrays and the states of a run are held; fewer where the lanes
// behind the last column of a row and of the last wave would be more than a seventh of all.
int memory_width(const dl_memory_shape* s, int most) {
    auto lanes = [&](int V) { return ceil_div(s->N * ceil_div(s->D, V), 64) * 64 * V; };
    int V = most;
    while (V > 1 && (V > s->D || lanes(V) * 7 > lanes(1) * 8)) V /= 2;
    return V;
}
int widest_forward(int dtype) { return dtype == DL_F32 ? 2 : 4; }
int widest_back(int dtype) { return dtype == DL_F32 ? 1 : 2; }

// With a wave for every SIMD unit of the chip (1024) a wave runs through all of time.
form memory_form(const dl_memory_shape* s, int V) {
    form f{V, 1, 1, ceil_div(s->N * ceil_div(s->D, V), 64)};
    const int64_t runs = ceil_div(s->T, dlm::MARK);
    if (f.blocks >= 1024) return f;
    while (f.W < runs && f.W < dlm::WAVES) f.W *= 2;
    f.chunks = ceil_div(runs, f.W);
    return f;
}
// The form with the widest loads of its kernel.  The kernels that share the time axis hold a whole run in registers, and wait: four
// bytes there, for twice the waves (128 x 128 x 512 bf16: 17.4 instead of 18.0 us).
form memory_plan(const dl_memory_shape* s, int most) {
    form f = memory_form(s, memory_width(s, most));
    const int narrow = 4 / elem_bytes(s->dtype);
    return f.W > 1 && f.V > narrow ? memory_form(s, memory_width(s, narrow)) : f;
}
// A chain: its ticket, a link of two floats per chunk and column, a value per group of chunks.
int64_t chain_words(const dl_memory_shape* s, const form& f) { return (f.chunks + ceil_div(f.chunks, dlm::GROUP)) * s->N * s->D; }
int64_t chain_bytes(const dl_memory_shape* s, const form& f) { return f.chunks > 1 ? 64 + chain_words(s, f) * 8 : 0; }

dlm::chain start_chain(const dl_memory_shape* s, const form& f, void* workspace, hipStream_t st) {
    uint64_t* links = (uint64_t*)((char*)workspace + 64);
    const dlm::chain ch{(uint32_t*)workspace, links, links + f.chunks * s->N * s->D, (uint32_t)f.blocks};
    const int64_t words = chain_words(s, f);
    dlm::k_memory_unlink<<<(unsigned)std::min<int64_t>(1024, ceil_div(words, 1024)), 256, 0, st>>>(ch, words);
    return ch;
}

dlm::shape device_shape(const dl_memory_shape* s, const form& f) {
    return dlm::shape{s->N, s->D, s->x_t, s->x_n, s->gate_t, s->gate_n, s->starts_t, s->starts_n, s->grad_t, s->grad_n, (int32_t)s->T, (int32_t)f.chunks};
}

template <int N> struct Int { static constexpr int value = N; };
template <typename F> void with_waves(int W, F&& f) {          // more than one
    if (W == 8) f(Int<8>()); else if (W == 4) f(Int<4>()); else f(Int<2>());
}
template <int MOST, typename F> void with_width(int V, F&& f) {
    if constexpr (MOST >= 4) if (V == 4) return f(Int<4>());
    if constexpr (MOST >= 2) if (V == 2) return f(Int<2>());
    f(Int<1>());
}
template <typename E> constexpr int widest() { return sizeof(E) == 4 ? 2 : 4; }
template <typename F> void with_type(int dtype, F&& f) {
    if (dtype == DL_F32) f(float{}); else if (dtype == DL_BF16) f(__bf16{}); else f(_Float16{});
}

// ---- orthogonalised updates ----
const char* orth_shape_error(const dl_orth_shape* s) {
    if (!s) return "shape must not be NULL";
    for (int t : {s->grad_type, s->weight_type, s->out_type})
        if (t != DL_F32 && t != DL_BF16 && t != DL_F16) return "unknown type";
    if (s->reserved != 0) return "reserved must be 0";
    if (s->batch < 0 || s->rows < 0 || s->cols < 0) return "batch, rows and cols must not be negative";
    if (s->batch > 65535 || s->rows > (1 << 20) || s->cols > (1 << 20)) return "more than 65535 matrices, or a side above 2^20";
    if (s->rows * s->cols > ((int64_t)1 << 32)) return "a matrix of more than 2^32 elements";
    if (s->steps < 1 || s->steps > 100) return "steps must be 1 .. 100";
    for (int64_t st : {s->grad_b, s->grad_r, s->momentum_b, s->momentum_r, s->momentum_out_b, s->momentum_out_r, s->weight_b, s->weight_r, s->out_b, s->out_r})
        if (st < 0) return "negative strides";
    return nullptr;
}

// What the planes hold (dl_orth.hpp) times 2^10, and float16 only up to 65504: X, A = X X' and Q = a I + b A + c A A of every step.  An entry is at most
// the largest singular value.  X's lie in [0, 1] at first, and a step takes s to s q(s^2), q(u) = a + b u + c u^2; the largest of either is at an end of
// the interval or where a derivative is zero.
constexpr double MOST = 60.0;
bool coefficients_hold(int steps, double a, double b, double c) {
    auto q = [&](double u) { return a + u * (b + u * c); };
    double s = 1.0;          // the largest singular value there may be
    for (int k = 0; k < steps; ++k) {
        const double u1 = s * s;
        auto inside = [&](double u) { return u > 0.0 && u < u1; };
        double most_q = std::max(std::fabs(q(0.0)), std::fabs(q(u1)));
        const double top = -b / (2.0 * c);
        if (inside(top)) most_q = std::max(most_q, std::fabs(q(top)));
        if (!(s < MOST && u1 < MOST && most_q < MOST)) return false;
        double next = s * std::fabs(q(u1));
        const double root = 9.0 * b * b - 20.0 * a * c;          // a + 3 b u + 5 c u^2 = 0
        if (root >= 0.0) {
            const double t = -0.5 * (3.0 * b + std::copysign(std::sqrt(root), b));
            for (double u : {t / (5.0 * c), a / t})
                if (inside(u)) next = std::max(next, std::sqrt(u) * std::fabs(q(u)));
        }
        s = next;
    }
    return true;
}

struct orth_form {
    dlo::plan p;
    int tile;
    bool turned, small, slab, gram_direct, poly_direct;          // direct: k_orth_direct for this product
    int64_t slab_rows, slab_cols, n_slabs;    // 16 rows, columns and number of slabs
    int64_t splits, counters;                 // of a Gram tile along its sum, and the counters of all tiles
    int64_t head, x_bytes, a_bytes, bytes;    // the workspace: partials, counters and split sums (together head), XR, XC, XC', A, Q of the whole batch
};

constexpr int64_t DIRECT = (int64_t)800 * 800 * 800;

orth_form orth_plan(const dl_orth_shape* s) {
    orth_form f;
    f.turned = s->rows > s->cols;
    f.p.m = (int32_t)std::min(s->rows, s->cols);
    f.p.n = (int32_t)std::max(s->rows, s->cols);
    f.small = f.p.n <= (f.p.m <= 16 ? 1024 : f.p.m <= 32 ? 512 : f.p.m <= 64 ? 256 : 0);          // what a workgroup's LDS and registers hold
    // Short sides of up to 64: a slab of 512 columns (up to 32 rows) or 256 per workgroup; from 256 slabs on the sums over them weigh more
    // than the launches they save (and the products of up to 16 rows are those of 22-bit operands, as for larger matrices).
    f.slab_rows = f.p.m <= 16 ? 1 : f.p.m <= 32 ? 2 : 4;
    f.slab_cols = f.slab_rows == 4 ? 256 : 512;
    f.n_slabs = ceil_div(f.p.n, f.slab_cols);
    f.slab = !f.small && f.p.m <= 64 && f.n_slabs < 256;
    const int64_t m32 = ceil_div(f.p.m, 32) * 32, n32 = ceil_div(f.p.n, 32) * 32;
    // Whatever sets the order of a matrix's sums (tile, direct or staged, splits) follows from that matrix alone, never from how many come
    // with it: a matrix has the same result, bit for bit, by itself and in any stack.
    // What that costs where a rule on the whole stack would have taken the staged kernels: 16 x 512 x 512 404 instead of 359 us, 64 x 512 x
    // 512 1515 instead of 1154, 8 x 100 x 8000 509 instead of 262; 4 x 700 x 700 gains, 241 instead of 274.
    f.tile = m32 * m32 * n32 <= DIRECT ? 32 : 128;
    f.p.mp = (int32_t)(ceil_div(f.p.m, f.tile) * f.tile);
    f.p.np = (int32_t)(ceil_div(f.p.n, f.tile) * f.tile);
    f.p.x_size = (int64_t)f.p.mp * f.p.np * 2;
    f.p.a_size = (int64_t)f.p.mp * f.p.mp * 2;
    f.p.partials = (int32_t)std::min<int64_t>(1024, ceil_div(s->rows * s->cols, 4096));
    f.x_bytes = s->batch * f.p.x_size * 2;
    f.a_bytes = s->batch * f.p.a_size * 2;
    // Of a product with few tiles in the staged kernels the direct one may be the faster: 0.27 us a step of 64 x 64 tiles against 64 rows
    // from the caches for every 32 x 32 tile, at 10 TB/s, and 3 us more where the sum is split.
    auto direct = [&](int64_t k) {
        const int64_t t64 = f.p.mp / 64 * (f.p.mp / 64 + 1) / 2, t32 = f.p.mp / 32 * (f.p.mp / 32 + 1) / 2;
        return f.tile == 32 || (double)ceil_div(t64, 512) * (double)(k / 32) * 0.27 > (double)t32 * 64 * (double)k * 4 * 1e-7 + 3;
    };
    f.gram_direct = direct(f.p.np);
    f.poly_direct = direct(f.p.mp);
    // A workgroup per CU and two steps for each of its eight waves; not worth the way through memory below some hundred steps.
    const int64_t tri = f.p.mp / 32 * (f.p.mp / 32 + 1) / 2, steps = f.p.np / 32;
    f.splits = f.gram_direct && steps >= 128 ? std::max<int64_t>(1, std::min<int64_t>({ceil_div(256, tri), steps / 16, 64})) : 1;
    f.counters = f.splits > 1 ? s->batch * tri : 0;
    f.head = ceil_div(s->batch * f.p.partials * 8 + f.counters * 4, 256) * 256;
    if (f.slab) {          // the head, X and two sets of sums
        f.x_bytes = s->batch * f.n_slabs * f.slab_rows * 16 * f.slab_cols * 4;
        f.a_bytes = s->batch * f.n_slabs * (f.slab_rows * (f.slab_rows + 1) / 2) * 1024;
        f.bytes = f.head + f.x_bytes + 2 * f.a_bytes;
        return f;
    }
    f.bytes = f.head + f.counters * f.splits * 4096 + 3 * f.x_bytes + 2 * f.a_bytes;
    return f;
}

// How many of `tiles` per matrix run whole when `slots` of them fill the chip: a last round of less than two thirds is cut up.
int32_t whole_tiles(int64_t tiles, int64_t batch, int64_t slots) {
    const int64_t rest = tiles * batch % slots;
    return rest * 3 >= slots * 2 ? (int32_t)tiles : (int32_t)(tiles - std::min(tiles, ceil_div(rest, batch)));
}

// Tiles of 256 x 128 (a CU each) where they come to at least nine tenths of a round of whole ones and what is left in 64 x 64 to one
// round at most, else of 128 x 128 (two to a CU).  4096 x 8192 x 4096: 610 instead of 652 us; 2 x 1031 x 4099 x 1031, where 328 of
// 64 x 64 would be left: 71 and 68 us.
template <int TILE, int MODE> void launch_product(dlo::product p, int64_t tiles, int64_t batch, const orth_form& f, hipStream_t st) {
    const dlo::plan& q = f.p;
    if (TILE == 32 || (MODE == dlo::GRAM && f.gram_direct) || (MODE == dlo::POLY && f.poly_direct)) {
        if (TILE != 32) tiles = (int64_t)(q.mp / 32) * (q.mp / 32 + 1) / 2;
        dlo::k_orth_direct<MODE><<<dim3((unsigned)(MODE == dlo::GRAM ? tiles * p.splits : tiles), 1, (unsigned)batch), 512, 0, st>>>(p);
    } else if constexpr (TILE != 32) {
        constexpr bool half = MODE == dlo::GRAM || MODE == dlo::POLY;
        const int64_t wi = q.mp / 256, wj = q.np / 128, wide = half ? wi * (wi + 1) : wi * wj, whole = whole_tiles(wide, batch, 256);
        const int64_t left = (wide - whole) * 8 + (q.mp % 256 ? 2 * (half ? q.mp / 64 : q.np / 64) : 0);
        if (whole * batch >= 230 && left * batch <= 256) {
            p.tiles = (int32_t)wide; p.whole = (int32_t)whole;
            p.tiles_i = (int32_t)wi; p.tiles_j = (int32_t)wj;
            return dlo::k_orth_wide<MODE><<<dim3((unsigned)(whole + left), 1, (unsigned)batch), 256, 0, st>>>(p);
        }
        p.tiles = (int32_t)tiles; p.whole = whole_tiles(tiles, batch, 512);
        dlo::k_orth_product<MODE><<<dim3((unsigned)(p.whole + (tiles - p.whole) * 4), 1, (unsigned)batch), 256, 0, st>>>(p);
    }
}

template <int TILE> void launch_steps(const dl_orth_shape* s, const orth_form& f, dlo::product last, char* work, hipStream_t st) {
    _Float16* xr = (_Float16*)work;
    _Float16* xc[2] = {(_Float16*)(work + f.x_bytes), (_Float16*)(work + 2 * f.x_bytes)};
    _Float16* A = (_Float16*)(work + 3 * f.x_bytes);
    _Float16* Q = (_Float16*)(work + 3 * f.x_bytes + f.a_bytes);
    const int64_t ti = f.p.mp / TILE, tj = f.p.np / TILE, tri = ti * (ti + 1) / 2;
    const int32_t km = f.p.mp / 32, kn = f.p.np / 32;
    for (int k = 0; k < s->steps; ++k) {
        const bool end = k + 1 == s->steps;
        dlo::product p = last;
        p.P = p.Q = xr; p.P_b = p.Q_b = f.p.x_size; p.kb = kn;
        p.out0 = A; p.out0_b = f.p.a_size; p.out0_kb = km;
        launch_product<TILE, dlo::GRAM>(p, tri, s->batch, f, st);
        p.P = p.Q = A; p.P_b = p.Q_b = f.p.a_size; p.kb = km;
        p.A = A; p.out0 = Q;
        launch_product<TILE, dlo::POLY>(p, tri, s->batch, f, st);
        p.P = Q; p.Q = xc[k & 1]; p.Q_b = f.p.x_size;
        p.tiles_i = (int32_t)ti; p.tiles_j = (int32_t)tj;
        p.out0 = xr; p.out0_b = f.p.x_size; p.out0_kb = kn;
        p.out1 = xc[(k + 1) & 1]; p.out1_b = f.p.x_size; p.out1_kb = km;
        if (end) launch_product<TILE, dlo::LAST>(p, ti * tj, s->batch, f, st); else launch_product<TILE, dlo::STEP>(p, ti * tj, s->batch, f, st);
    }
}

}  // namespace

extern "C" {

const char* dl_learner_last_error(void) { return g_err.c_str(); }
int dl_learner_abi_version(void) { return DL_LEARNER_ABI_VERSION; }

int64_t dl_memory_workspace_bytes(const dl_memory_shape* s) {
    if (const char* e = memory_shape_error(s)) return fail(DL_E_INVAL, e);
    if (s->T == 0 || s->N == 0 || s->D == 0) return 0;
    int64_t most = 0;
    for (int V : {widest_forward(s->dtype), widest_back(s->dtype)}) most = std::max(most, chain_bytes(s, memory_plan(s, V)));
    return most;
}

int dl_memory_forward(const dl_memory_shape* s, const void* x, const void* gate, const uint8_t* starts, const float* state, void* h, float* state_out, float* marks, void* workspace, void* stream) {
    if (const char* e = memory_shape_error(s)) return fail(DL_E_INVAL, e);
    if (s->N == 0 || s->D == 0) return DL_OK;
    if (s->T == 0) return fail(DL_E_INVAL, "dl_memory_forward: T = 0 (there is no step: the state stays as it is)");
    if (!x || !gate || !h) return fail(DL_E_INVAL, "dl_memory_forward: x, gate and h must not be NULL");
    if (state && state == state_out) return fail(DL_E_INVAL, "dl_memory_forward: state_out may not be state");
    const form f = memory_plan(s, widest_forward(s->dtype));
    if (f.chunks > 1 && !workspace) return fail(DL_E_INVAL, "dl_memory_forward: workspace must not be NULL (dl_memory_workspace_bytes)");
    if (!aligned(workspace, 16)) return fail(DL_E_INVAL, "dl_memory_forward: workspace must be aligned to 16 bytes");
    if (!fits(f.blocks * f.chunks, 64 * f.W)) return fail(DL_E_INVAL, "dl_memory_forward: T * N * D too large");
    const dlm::shape d = device_shape(s, f);
    const unsigned grid = (unsigned)(f.blocks * f.chunks);
    hipStream_t st = (hipStream_t)stream;
    with_type(s->dtype, [&](auto e) { with_width<widest<decltype(e)>()>(f.V, [&](auto v) {
        using E = decltype(e);
        constexpr int V = decltype(v)::value;
        if (f.W == 1) {
            dlm::k_memory_run<E, V><<<grid, 64, 0, st>>>(d, (const E*)x, (const E*)gate, starts, state, (E*)h, state_out, marks);
        } else if constexpr (V * sizeof(E) <= 4) {
            if (f.chunks > 1) {
                const dlm::chain ch = start_chain(s, f, workspace, st);
                dlm::k_memory_short<E, V, dlm::WAVES, true><<<grid, 64 * dlm::WAVES, 0, st>>>(d, ch, (const E*)x, (const E*)gate, starts, state, (E*)h, state_out, marks);
            } else with_waves(f.W, [&](auto w) {
                constexpr int W = decltype(w)::value;
                dlm::k_memory_short<E, V, W, false><<<grid, 64 * W, 0, st>>>(d, dlm::chain{}, (const E*)x, (const E*)gate, starts, state, (E*)h, state_out, marks);
            });
        }
    }); });
    return launched("dl_memory_forward");
}

int dl_memory_backward(const dl_memory_shape* s, const void* x, const void* gate, const uint8_t* starts, const float* marks, const void* grad_h, const float* grad_state, void* dx, void* dgate,
                       float* dstate, void* workspace, void* stream) {
    if (const char* e = memory_shape_error(s)) return fail(DL_E_INVAL, e);
    if (s->N == 0 || s->D == 0) return DL_OK;
    if (s->T == 0) return fail(DL_E_INVAL, "dl_memory_backward: T = 0 (there is no step: the gradient of the state is grad_state)");
    if (!x || !gate || !marks || !dx || !dgate) return fail(DL_E_INVAL, "dl_memory_backward: x, gate, marks, dx and dgate must not be NULL");
    if (grad_state && grad_state == dstate) return fail(DL_E_INVAL, "dl_memory_backward: dstate may not be grad_state");
    const form f = memory_plan(s, widest_back(s->dtype));
    if (f.chunks > 1 && !workspace) return fail(DL_E_INVAL, "dl_memory_backward: workspace must not be NULL (dl_memory_workspace_bytes)");
    if (!aligned(workspace, 16)) return fail(DL_E_INVAL, "dl_memory_backward: workspace must be aligned to 16 bytes");
    if (!fits(f.blocks * f.chunks, 64 * f.W)) return fail(DL_E_INVAL, "dl_memory_backward: T * N * D too large");
    const dlm::shape d = device_shape(s, f);
    const unsigned grid = (unsigned)(f.blocks * f.chunks);
    hipStream_t st = (hipStream_t)stream;
    with_type(s->dtype, [&](auto e) { with_width<widest<decltype(e)>() / 2>(f.V, [&](auto v) {
        using E = decltype(e);
        constexpr int V = decltype(v)::value;
        if (f.W == 1) {
            dlm::k_memory_run_back<E, V><<<grid, 64, 0, st>>>(d, (const E*)x, (const E*)gate, starts, marks, (const E*)grad_h, grad_state, (E*)dx, (E*)dgate, dstate);
        } else if (f.chunks > 1) {
            const dlm::chain ch = start_chain(s, f, workspace, st);
            dlm::k_memory_short_back<E, V, dlm::WAVES, true><<<grid, 64 * dlm::WAVES, 0, st>>>(d, ch, (const E*)x, (const E*)gate, starts, marks, (const E*)grad_h, grad_state, (E*)dx, (E*)dgate, dstate);
        } else with_waves(f.W, [&](auto w) {
            constexpr int W = decltype(w)::value;
            dlm::k_memory_short_back<E, V, W, false><<<grid, 64 * W, 0, st>>>(d, dlm::chain{}, (const E*)x, (const E*)gate, starts, marks, (const E*)grad_h, grad_state, (E*)dx, (E*)dgate, dstate);
        });
    }); });
    return launched("dl_memory_backward");
}

int dl_memory_step(const dl_memory_shape* s, const void* x, const void* gate, const uint8_t* starts, const float* state, void* h, float* state_out, void* stream) {
    if (const char* e = memory_shape_error(s)) return fail(DL_E_INVAL, e);
    if (s->T != 1) return fail(DL_E_INVAL, "dl_memory_step: T must be 1");
    if (s->N == 0 || s->D == 0) return DL_OK;
    if (!x || !gate || !h || !state_out) return fail(DL_E_INVAL, "dl_memory_step: x, gate, h and state_out must not be NULL");
    int V = widest_forward(s->dtype);
    while (s->D % V) V /= 2;
    const int64_t blocks = ceil_div(s->N * (s->D / V), 256);
    if (!fits(blocks, 256)) return fail(DL_E_INVAL, "dl_memory_step: N * D too large");
    with_type(s->dtype, [&](auto e) { with_width<widest<decltype(e)>()>(V, [&](auto v) {
        using E = decltype(e);
        constexpr int V_ = decltype(v)::value;
        dlm::k_memory_step<E, V_><<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(s->N, s->D, s->x_n, s->gate_n, s->starts_n, (const E*)x, (const E*)gate, starts, state, (E*)h, state_out);
    }); });
    return launched("dl_memory_step");
}

int dl_orth_check_coefficients(int32_t steps, double a, double b, double c) {
    if (steps < 1 || steps > 100) return fail(DL_E_INVAL, "steps must be 1 .. 100");
    if (!coefficients_hold(steps, a, b, c)) return fail(DL_E_INVAL, "the coefficients let X, X X' or a I + b X X' + c (X X')^2 grow to 60 or more within these steps");
    return DL_OK;
}

int64_t dl_orth_workspace_bytes(const dl_orth_shape* s) {
    if (const char* e = orth_shape_error(s)) return fail(DL_E_INVAL, e);
    if (s->batch == 0 || s->rows == 0 || s->cols == 0) return 0;
    const orth_form f = orth_plan(s);
    return f.small ? 0 : f.bytes;
}

int dl_orth_update(const dl_orth_shape* s, const void* grad, const float* momentum, float* momentum_out, const void* weight, void* out, void* workspace, void* stream) {
    if (const char* e = orth_shape_error(s)) return fail(DL_E_INVAL, e);
    if (s->batch == 0 || s->rows == 0 || s->cols == 0) return DL_OK;
    if (const int e = dl_orth_check_coefficients(s->steps, s->a, s->b, s->c)) return e;
    if (!grad || !out) return fail(DL_E_INVAL, "dl_orth_update: grad and out must not be NULL");
    if (!momentum != !momentum_out) return fail(DL_E_INVAL, "dl_orth_update: momentum and momentum_out must be given together");
    if (dl_orth_workspace_bytes(s) > 0 && !workspace) return fail(DL_E_INVAL, "dl_orth_update: workspace must not be NULL (dl_orth_workspace_bytes)");
    if (!aligned(workspace, 16)) return fail(DL_E_INVAL, "dl_orth_update: workspace must be aligned to 16 bytes");
    const orth_form f = orth_plan(s);
    hipStream_t st = (hipStream_t)stream;
    const bool flat = s->grad_r == s->cols && (!momentum || (s->momentum_r == s->cols && s->momentum_out_r == s->cols));          // one row as good as many
    const dlo::source src{grad, s->grad_type, momentum, momentum_out, (float)s->beta, s->nesterov, s->grad_b, s->grad_r, s->momentum_b, s->momentum_r, s->momentum_out_b, s->momentum_out_r};
    const dlo::small sp{src, f.p.m, f.p.n, s->steps, f.turned, flat && (!weight || s->weight_r == s->cols) && s->out_r == s->cols, (float)s->a, (float)s->b, (float)s->c,
                        out, weight, s->out_type, s->weight_type, s->out_b, s->out_r, s->weight_b, s->weight_r, (float)s->weight_keep, (float)s->gain};
    if (f.small) {
        const unsigned batch = (unsigned)s->batch;
        if (f.p.m > 32) dlo::k_orth_small<4, 2><<<batch, 512, 0, st>>>(sp);
        else if (f.p.m <= 16 && f.p.n <= 256) dlo::k_orth_small<1, 2><<<batch, 512, 0, st>>>(sp);
        else if (f.p.m <= 16 && f.p.n <= 512) dlo::k_orth_small<1, 4><<<batch, 512, 0, st>>>(sp);
        else if (f.p.m <= 16) dlo::k_orth_small<1, 8><<<batch, 512, 0, st>>>(sp);
        else if (f.p.n <= 256) dlo::k_orth_small<2, 2><<<batch, 512, 0, st>>>(sp);
        else dlo::k_orth_small<2, 4><<<batch, 512, 0, st>>>(sp);
        return launched("dl_orth_update");
    }
    double* partials = (double*)workspace;
    uint32_t* counters = (uint32_t*)(partials + s->batch * f.p.partials);
    float* parts = (float*)((char*)workspace + f.head);
    char* work = (char*)parts + f.counters * f.splits * 4096;
    dlo::k_orth_norm<<<dim3((unsigned)f.p.partials, (unsigned)s->batch), 256, 0, st>>>(src, flat ? 1 : s->rows, flat ? s->rows * s->cols : s->cols, partials, counters, (int)f.counters);
    if (f.slab) {
        char* at = (char*)workspace + f.head;
        dlo::slabs sl{partials, f.p.partials, (float*)at, {(float*)(at + f.x_bytes), (float*)(at + f.x_bytes + f.a_bytes)}, 0};
        dlo::small p = sp;
        p.flat = f.turned && sp.flat;          // (a slab of the caller's rows is one piece, one of columns is not)
        const dim3 grid((unsigned)s->batch, (unsigned)f.n_slabs);
        for (; sl.step <= s->steps; ++sl.step) {
            if (f.slab_rows == 1) dlo::k_orth_slab<1, 4><<<grid, 512, 0, st>>>(p, sl);
            else if (f.slab_rows == 2) dlo::k_orth_slab<2, 4><<<grid, 512, 0, st>>>(p, sl);
            else dlo::k_orth_slab<4, 2><<<grid, 512, 0, st>>>(p, sl);
        }
        return launched("dl_orth_update");
    }
    dlo::k_orth_load<<<dim3((unsigned)ceil_div(f.p.np, 64), (unsigned)ceil_div(f.p.mp, 64), (unsigned)s->batch), 256, 0, st>>>(src, f.p, f.turned, partials, (_Float16*)work, (_Float16*)(work + f.x_bytes));
    dlo::product p{};
    p.a = (float)s->a; p.b = (float)s->b; p.c = (float)s->c;
    p.out = out; p.w = weight; p.out_type = s->out_type; p.w_type = s->weight_type;
    p.out_at = f.turned ? dlo::matrix{s->out_b, 1, s->out_r} : dlo::matrix{s->out_b, s->out_r, 1};
    p.w_at = f.turned ? dlo::matrix{s->weight_b, 1, s->weight_r} : dlo::matrix{s->weight_b, s->weight_r, 1};
    p.splits = (int32_t)f.splits; p.parts = parts; p.arrived = counters;
    p.keep = (float)s->weight_keep; p.gain = (float)s->gain;
    p.m = f.p.m; p.n = f.p.n;
    if (f.tile == 32) launch_steps<32>(s, f, p, work, st); else launch_steps<128>(s, f, p, work, st);
    return launched("dl_orth_update");
}

}  // extern "C"
