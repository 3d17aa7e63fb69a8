// dl_memory.hpp -- the gated memory of a recurrent policy over a rollout: forward, gradients, one control step.
//
//     a = sigmoid(g), s = 1 - a:      h[t] = a h' + s x[t],   h' = start ? 0 : h[t-1]
//     l[t] = dh[t] + c[t+1],  c[t] = start ? 0 : a l[t]:      dx = s l,   dg = (h' - x) a s l,   dstate = c[0]
//
// Bound by memory (three elements moved per step forward, five backward) with the arithmetic, 20 to 40 operations per element, close
// behind.  A wave takes 64 x V columns through time, MARK steps (a run) in registers and the loads of the next ones under way.
// Three forms, by the number of such waves ("blocks") and of steps:
//   whole   enough blocks for the chip: a wave runs through all of time, every element is loaded once;
//   short   few blocks, at most eight runs: the waves of a workgroup take a run each, reduce it to its affine map, exchange the maps
//           through LDS and finish their steps from the registers: every element is loaded once here too;
//   chain   few blocks, more runs: a row of such workgroups along time.  Each leaves its map in memory as soon as it has it and picks
//           up those before it while its own elements wait in registers: once again every element is loaded once.
//
// Rounding.  The smaller of a and s is computed as e / (1 + e), e = exp(-|g|), and both products go through it:
//     g >= 0:  h = h' + s (x - h'),  c = l - s l        g < 0:  h = x + a (h' - x),  c = a l
// so that a long memory (s small) loses nothing to the rounding of a = 1 - s, and a closed gate gives x exactly.  The differences
// are taken of halves: x and h of up to the largest number are well.
//
// Columns.  A lane takes V neighbouring channels with one load (4 or 8 bytes, any alignment); where V does not divide D the last
// lane of a row moves back, and two lanes compute, and write, the same values.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

namespace dlm {

constexpr int MARK = 16;          // steps of a wave's run, and between two saved states
constexpr int WAVES = 8;          // waves of a chain's workgroup, a run each

template <typename E, int V> struct vec { typedef E type __attribute__((ext_vector_type(V), aligned(sizeof(E)))); };
template <typename E> struct vec<E, 1> { typedef E type; };
template <typename E, int V> using vec_t = typename vec<E, V>::type;

template <typename E, int V> __device__ __forceinline__ float get(const vec_t<E, V>& v, int i) {
    if constexpr (V == 1) return (float)v; else return (float)v[i];
}
template <typename E, int V> __device__ __forceinline__ void put(vec_t<E, V>& v, int i, float f) {
    // float16: rounded from the 32-bit value everywhere, not in one kernel by a product-sum that rounds to 16 bits at once
    if constexpr (std::is_same<E, _Float16>::value) asm("" : "+v"(f));
    if constexpr (V == 1) v = (E)f; else v[i] = (E)f;
}

struct shape {
    int64_t N, D;
    int64_t x_t, x_n, gate_t, gate_n, starts_t, starts_n, grad_t, grad_n;
    int32_t T, chunks;            // steps; workgroups along time
};

// min(a, s) with the sign of the gate.
__device__ __forceinline__ float gate_of(float g) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269504f);
    return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), g);
}
__device__ __forceinline__ bool keeps(float m) { return !(__float_as_uint(m) >> 31); }          // s is the smaller one
// f (x - h) + rest.  The difference may be beyond the largest number where the product is not, so it is taken of halves (2 f is a number: f is a gate
// or a quarter of a gradient at most); not with x in float16, from which no float32 is further away than that (100003 x 333: 105 us, of halves 113).
template <typename E> constexpr bool wide = !std::is_same<E, _Float16>::value;
template <typename E> __device__ __forceinline__ float times_apart(float f, float x, float h, float rest) {
    return wide<E> ? fmaf(f + f, fmaf(-0.5f, h, 0.5f * x), rest) : fmaf(f, x - h, rest);
}
// one step of the state
template <typename E> __device__ __forceinline__ float step_of(float m, float x, float h) {
    return times_apart<E>(m, x, h, keeps(m) ? h : x);           // (m < 0: x + |m| (h - x) = x + m (x - h))
}
// one step of a product of a: l -> a l
__device__ __forceinline__ float decay_of(float m, float l) {
    const float w = m * l;
    return keeps(m) ? l - w : -w;
}

// The map h -> a h + b of a run, a = the product of its steps'.  Like a step it is held by the smaller of a and p = 1 - a: m = p
// where p <= 1/2, else -a; so a product over thousands of open gates is as exact as its steps.  BEGUN: an episode began inside
// the run, nothing before it counts, not even a NaN.
constexpr float BEGUN = 2.0f;
struct factor {
    float a = 1.0f, p = 0.0f;
    __device__ __forceinline__ void step(float m) {
        const float w = fabsf(m) * a, o = a - w;
        p += keeps(m) ? w : o;
        a = keeps(m) ? o : w;
    }
    __device__ __forceinline__ float held(bool begun) const { return begun ? BEGUN : p <= 0.5f ? p : -a; }          // (a NaN stays one)
};
__device__ __forceinline__ float apply(float m, float b, float h) { return m > 1.0f ? b : decay_of(m, h) + b; }
// Of states: the sum of two shares of finite values lies between them, but may be rounded past the largest number (not with x in float16, whose
// share is lost next to such a state's).
__device__ __forceinline__ float apply_state(float m, float b, float h) {
    const float r = apply(m, b, h);
    return __builtin_isinf(r) && __builtin_isfinite(b) && __builtin_isfinite(h) ? copysignf(__FLT_MAX__, r) : r;
}
__device__ __forceinline__ float after(float m, float n) {          // m, then n
    if (m > 1.0f || n > 1.0f) return BEGUN;
    factor f;
    f.step(m); f.step(n);
    return f.held(false);
}

__device__ __forceinline__ int64_t uniform(int64_t v) {          // the same in all lanes: into scalar registers
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// Where a lane's columns lie.  Rows are addressed as a pointer of the workgroup (scalar registers) at channel 0 of its first walker,
// n0, plus 32 bits of a lane; the host refuses strides for which 64 walkers are further apart than that.
template <int V> struct columns {
    int64_t n0;
    uint32_t dn, d;               // walkers after n0, channel
    bool valid, few;              // few: the wave spans at most four walkers
    __device__ columns(int64_t N, int64_t D, uint32_t block = blockIdx.x) {
        const int64_t per = (D + V - 1) / V;
        const int64_t q0 = (int64_t)block * 64, q = q0 + (threadIdx.x & 63);
        n0 = uniform(q0 / per);
        valid = q < N * per;
        dn = valid ? (uint32_t)(q / per - n0) : 0;
        d = valid ? (uint32_t)min((q - (n0 + dn) * per) * V, D - V) : 0;
        few = per >= 32;
    }
    template <typename E> __device__ __forceinline__ uint32_t bytes(int64_t stride_n) const { return (dn * (uint32_t)stride_n + d) * (uint32_t)sizeof(E); }
};
// base in scalar registers, kept there: no 64-bit addition per lane and access
#define DLM_GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ __forceinline__ T load_at(const void* base, uint32_t bytes) {
    const DLM_GLOBAL char* p = (const DLM_GLOBAL char*)base;
    asm("" : "+s"(p));
    return *(const DLM_GLOBAL T*)(p + bytes);
}
template <typename T> __device__ __forceinline__ void store_at(void* base, uint32_t bytes, const T& v) {
    DLM_GLOBAL char* p = (DLM_GLOBAL char*)base;
    asm("" : "+s"(p));
    *(DLM_GLOBAL T*)(p + bytes) = v;
}

// The value that enters the run of each wave from the maps of the waves before it (`before` of them, in the order of the
// recurrence), and the one behind the last.  STATE: of states that may reach the largest number.
template <int V, bool BACK, bool STATE>
__device__ __forceinline__ void join(const float (*la)[64 * V], const float (*lb)[64 * V], int lane, int waves, int before, const float (&carry)[V], float (&mine)[V], float (&next)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) next[v] = mine[v] = carry[v];
    for (int i = 0; i < waves; ++i) {
        const int w = BACK ? waves - 1 - i : i;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            next[v] = STATE ? apply_state(la[w][v * 64 + lane], lb[w][v * 64 + lane], next[v]) : apply(la[w][v * 64 + lane], lb[w][v * 64 + lane], next[v]);
            if (i + 1 == before) mine[v] = next[v];
        }
    }
}

template <int V> __device__ __forceinline__ void load_floats(float (&to)[V], const float* base, uint32_t bytes) {
    const vec_t<float, V> f = load_at<vec_t<float, V>>(base, bytes);
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = get<float, V>(f, v);
}
template <int V> __device__ __forceinline__ void store_floats(float* base, uint32_t bytes, const float (&from)[V]) {
    vec_t<float, V> f;
#pragma unroll
    for (int v = 0; v < V; ++v) put<float, V>(f, v, from[v]);
    store_at<vec_t<float, V>>(base, bytes, f);
}

// Between the passes over a run: the comparisons of the first are made again instead of being kept, a pair of scalar registers each.
template <int V> __device__ __forceinline__ void forget(float (&m)[MARK][V], uint32_t& begin) {
#pragma unroll
    for (int t = 0; t < MARK; ++t) {
#pragma unroll
        for (int v = 0; v < V; ++v) asm volatile("" : "+v"(m[t][v]));
    }
    asm volatile("" : "+v"(begin));
}

template <typename T> __device__ __forceinline__ void opaque(T& v) {
    if constexpr (sizeof(T) == 8) { uint64_t u = __builtin_bit_cast(uint64_t, v); asm volatile("" : "+v"(u)); v = __builtin_bit_cast(T, u); }
    else if constexpr (sizeof(T) == 4) { uint32_t u = __builtin_bit_cast(uint32_t, v); asm volatile("" : "+v"(u)); v = __builtin_bit_cast(T, u); }
    else { uint16_t u = __builtin_bit_cast(uint16_t, v); asm volatile("" : "+v"(u)); v = __builtin_bit_cast(T, u); }
}
// The scheduler would start all the steps of a run at once and keep their halves in registers: every few elements it may not look further.
template <int V> __device__ __forceinline__ void pause(int t) {
    if ((t + 1) * V % 8 == 0) __builtin_amdgcn_sched_barrier(0);
}

// Rows t0 .. t0 + R - 1 as they lie in memory.  Rows behind the end read the last one again.
template <typename E, int V, int R, bool X, bool G> struct rows {
    typedef vec_t<E, V> vec;
    vec x[R], g[R], d[R];
    uint32_t begin;               // bit t: an episode begins at row t
    uint8_t flag;                 // few walkers: lane 16 w + t looks at row t of walker n0 + w, for all

    __device__ __forceinline__ static void each(vec (&to)[R], const E* base, int64_t stride, uint32_t off, int len) {
        const E* p = base;
        if (len >= R) {
#pragma unroll
            for (int t = 0; t < R; ++t) { to[t] = load_at<vec>(p, off); p += stride; }
        } else {
#pragma unroll
            for (int t = 0; t < R; ++t) { to[t] = load_at<vec>(p, off); if (t + 1 < len) p += stride; }
        }
    }
    __device__ __forceinline__ void load(const shape& s, const columns<V>& c, int t0, int last, const E* x_, const E* g_, const E* d_, const uint8_t* b_) {
        const int len = max(0, min(R, last - t0));
        const int64_t from = min(t0, last - 1);
        if (X) each(x, x_ + from * s.x_t + c.n0 * s.x_n, s.x_t, c.template bytes<E>(s.x_n), len);
        each(g, g_ + from * s.gate_t + c.n0 * s.gate_n, s.gate_t, c.template bytes<E>(s.gate_n), len);
        if (G) {
            if (d_) each(d, d_ + from * s.grad_t + c.n0 * s.grad_n, s.grad_t, c.template bytes<E>(s.grad_n), len);
            else {
#pragma unroll
                for (int t = 0; t < R; ++t)
#pragma unroll
                    for (int v = 0; v < V; ++v) put<E, V>(d[t], v, 0.0f);
            }
        }
        begin = 0;
        flag = 0;
        if (b_) {
            const uint8_t* p = b_ + from * s.starts_t + c.n0 * s.starts_n;
            if (c.few) {
                const int t = threadIdx.x & 15, w = (threadIdx.x >> 4) & 3;
                if (t < len && c.n0 + w < s.N) flag = p[(int64_t)t * s.starts_t + (int64_t)w * s.starts_n];
            } else {
#pragma unroll
                for (int t = 0; t < R; ++t)
                    if (t < len) begin |= (uint32_t)(p[(int64_t)t * s.starts_t + (int64_t)c.dn * s.starts_n] != 0) << t;
            }
        }
    }
    // when the rows are needed
    __device__ __forceinline__ uint32_t begins(const columns<V>& c) const {
        return c.few ? (uint32_t)(__ballot(flag != 0) >> (16 * c.dn)) & 0xffffu : begin;
    }
    // As forget(): what was converted from the elements is converted again.
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int t = 0; t < R; ++t) { if (X) opaque(x[t]); if (G) opaque(d[t]); }
    }
};

struct yes { static constexpr bool value = true; };
struct no { static constexpr bool value = false; };

// ---- whole: a wave runs through all steps, half a run ahead with its loads --------------------------------------------------------------
// 512 x 4096 x 128 bf16 with marks: 1.68 GB in 355 us, 4.7 TB/s, what a large copy reaches; bound by memory.
template <typename E, int V>
__global__ __launch_bounds__(64) void k_memory_run(shape s, const E* __restrict__ x, const E* __restrict__ gate, const uint8_t* __restrict__ starts, const float* __restrict__ state,
                                                   E* __restrict__ h, float* __restrict__ state_out, float* __restrict__ marks) {
    typedef vec_t<E, V> vec;
    constexpr int R = MARK / 2;
    typedef rows<E, V, R, true, false> half;
    const columns<V> c(s.N, s.D);
    const int64_t plane = s.N * s.D, corner = c.n0 * s.D;
    const uint32_t elems = c.template bytes<E>(s.D), floats = c.template bytes<float>(s.D);
    float now[V];
#pragma unroll
    for (int v = 0; v < V; ++v) now[v] = 0.0f;
    if (state) load_floats<V>(now, state + corner, floats);
    auto steps = [&](const half& r, int t0, int len, auto all, uint32_t begin) {
        E* ph = h + (int64_t)t0 * plane + corner;
#pragma unroll
        for (int t = 0; t < R; ++t) {
            if (decltype(all)::value || t < len) {
                vec o;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (!decltype(all)::value) now[v] = (begin >> t) & 1 ? 0.0f : now[v];
                    now[v] = step_of<E>(gate_of(get<E, V>(r.g[t], v)), get<E, V>(r.x[t], v), now[v]);
                    put<E, V>(o, v, now[v]);
                }
                if (c.valid) store_at<vec>(ph, elems, o);
                ph += plane;
            }
        }
    };
    auto run = [&](const half& r, int t0) {          // whole and without a beginning, as nearly always, or not
        const int len = max(0, min(R, s.T - t0));
        const uint32_t begin = r.begins(c);
        if (len == R && __ballot(begin != 0) == 0) steps(r, t0, len, yes(), 0u); else steps(r, t0, len, no(), begin);
    };
    half p, q;
    p.load(s, c, 0, s.T, x, gate, nullptr, starts);
    for (int t0 = 0; t0 < s.T; t0 += MARK) {
        q.load(s, c, t0 + R, s.T, x, gate, nullptr, starts);
        if (marks && c.valid) store_floats<V>(marks + (int64_t)(t0 / MARK) * plane + corner, floats, now);
        run(p, t0);
        p.load(s, c, t0 + MARK, s.T, x, gate, nullptr, starts);
        run(q, t0 + R);
    }
    if (state_out && c.valid) store_floats<V>(state_out + corner, floats, now);
}

// ---- chain: the maps of workgroups on their way to later ones ---------------------------------------------------------------------------
// A link is the map (m, b) of a workgroup in one 64-bit word, written and read whole, so that there is nothing to order; EMPTY (no map
// has that m) until it is written.  Of every GROUP workgroups the last also leaves the value behind it, so that the next group starts
// from that and no workgroup joins more than GROUP - 1 links.  Workgroups take their place in the chain by a ticket, in the order in
// which they start: those a workgroup waits for have started before it, and wait only for earlier ones in turn, the first for nobody,
// so every wait ends.  What is joined, and in which order, does not depend on who comes late, nor do results.
constexpr int GROUP = 64;
constexpr uint32_t EMPTY = 0xffffffffu;
struct chain { uint32_t* ticket; uint64_t *links, *values; uint32_t blocks; };          // links: [chunks][N * D], values: [groups][N * D] (behind them)

__global__ __launch_bounds__(256) void k_memory_unlink(chain ch, int64_t words) {
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < words; e += (int64_t)gridDim.x * 256) ch.links[e] = ~0ull;
    if (blockIdx.x == 0 && threadIdx.x == 0) *ch.ticket = 0;
}

template <int V> __device__ __forceinline__ void link(uint64_t* at, const float (&m)[V], const float (&b)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const uint32_t lo = m[v] != m[v] ? 0x7fc00000u : __float_as_uint(m[v]);
        __hip_atomic_store(at + v, (uint64_t)__float_as_uint(b[v]) << 32 | lo, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
// m, b: joined with the links of the chunks first, first + way, .. (`count` of them)
template <int V, bool STATE> __device__ __forceinline__ void follow(const uint64_t* links, int64_t plane, int first, int way, int count, float (&m)[V], float (&b)[V]) {
    constexpr int AT_ONCE = 4;
    for (int i = 0; i < count; i += AT_ONCE) {
        uint64_t l[AT_ONCE][V];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) l[k][v] = __hip_atomic_load(links + (int64_t)(first + way * min(i + k, count - 1)) * plane + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (i + k >= count) break;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                while ((uint32_t)l[k][v] == EMPTY) {
                    __builtin_amdgcn_s_sleep(1);
                    l[k][v] = __hip_atomic_load(links + (int64_t)(first + way * (i + k)) * plane + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                const float n = __uint_as_float((uint32_t)l[k][v]), c = __uint_as_float((uint32_t)(l[k][v] >> 32));
                b[v] = STATE ? apply_state(n, c, b[v]) : apply(n, c, b[v]);
                m[v] = after(m[v], n);
            }
        }
    }
}
__device__ __forceinline__ uint32_t take_ticket(const chain& ch) {
    __shared__ uint32_t mine;
    if (threadIdx.x == 0) mine = __hip_atomic_fetch_add(ch.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane((int)mine);
}
// Leaves the workgroup's link (from its waves' maps la, lb) and finds the value that enters it; carry: the one that enters the chain.
template <int V, bool BACK, bool STATE>
__device__ __forceinline__ void pass_on(const chain& ch, int k, int chunks, int64_t plane, int64_t col, bool valid, int wave, int lane, const float (*la)[64 * V], const float (*lb)[64 * V],
                                        float (*lc)[64 * V], float (*ld)[64 * V], float (&carry)[V]) {
    const int order = BACK ? chunks - 1 - k : k, before = order % GROUP;
    float m[V], b[V], zero[V], mine[V], next[V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = b[v] = zero[v] = 0.0f;
    if (wave == 0 && before + 1 < GROUP && order + 1 < chunks) {          // (of the last one of a group nobody takes the link)
        join<V, BACK, STATE>(la, lb, lane, WAVES, 0, zero, mine, next);
        for (int w = 0; w < WAVES; ++w) {
#pragma unroll
            for (int v = 0; v < V; ++v) m[v] = after(m[v], la[w][v * 64 + lane]);
        }
        if (valid) link<V>(ch.links + (int64_t)k * plane + col, m, next);
    }
    if (before > 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) m[v] = b[v] = 0.0f;
        const int lo = before * wave / WAVES, hi = before * (wave + 1) / WAVES, way = BACK ? -1 : 1;
        follow<V, STATE>(ch.links + col, plane, k - way * (before - lo), way, hi - lo, m, b);
#pragma unroll
        for (int v = 0; v < V; ++v) { lc[wave][v * 64 + lane] = m[v]; ld[wave][v * 64 + lane] = b[v]; }
    }
    if (order >= GROUP) {
        const uint64_t* from = ch.values + (int64_t)(order / GROUP) * plane + col;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            uint64_t l = __hip_atomic_load(from + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            while ((uint32_t)(l >> 32) == EMPTY) {
                __builtin_amdgcn_s_sleep(1);
                l = __hip_atomic_load(from + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            carry[v] = __uint_as_float((uint32_t)l);
        }
    }
    if (before > 0) {
        __syncthreads();
        join<V, false, STATE>(lc, ld, lane, WAVES, 0, carry, mine, next);
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = next[v];
    }
}
// The value behind the last workgroup of a group.
template <int V, bool BACK> __device__ __forceinline__ void leave(const chain& ch, int k, int chunks, int64_t plane, int64_t col, bool valid, int wave, const float (&next)[V]) {
    const int order = BACK ? chunks - 1 - k : k;
    if (wave != 0 || !valid || (order + 1) % GROUP != 0 || order + 1 == chunks) return;
#pragma unroll
    for (int v = 0; v < V; ++v) __hip_atomic_store(ch.values + (int64_t)((order + 1) / GROUP) * plane + col + v, (uint64_t)__float_as_uint(next[v]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- short: W waves of a workgroup take one run each ----------------------------------------------------------------------------------
// 128 x 128 x 512 bf16: 52 MB in 17.6 us, 3.0 TB/s: a wave has one run, nothing is loaded meanwhile (vector units 0.69 busy).  Chains: 2048 x 8 x 512
// float32, 103 MB in 33 us, 3.1 TB/s; 3000 x 20 x 256 float32, 184 MB in 45 us, 4.1 TB/s; 100003 x 333 float16, 200 MB in 106 us, 1.9 TB/s:
// there 782 workgroups wait along one chain, in 13 groups that follow each other; waves wait 0.56 of their time, the vector units are 0.56 busy.
template <typename E, int V, int W, bool CHAIN>
__global__ __launch_bounds__(64 * W) void k_memory_short(shape s, chain ch, const E* __restrict__ x, const E* __restrict__ gate, const uint8_t* __restrict__ starts, const float* __restrict__ state,
                                                         E* __restrict__ h, float* __restrict__ state_out, float* __restrict__ marks) {
    typedef vec_t<E, V> vec;
    __shared__ float la[W][64 * V], lb[W][64 * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t place = CHAIN ? take_ticket(ch) : blockIdx.x, k = CHAIN ? place / ch.blocks : 0;
    const columns<V> c(s.N, s.D, CHAIN ? place - k * ch.blocks : place);
    const int64_t plane = s.N * s.D, corner = c.n0 * s.D;
    const uint32_t elems = c.template bytes<E>(s.D), floats = c.template bytes<float>(s.D);
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = 0.0f;
    if (state) load_floats<V>(carry, state + corner, floats);
    const int t0 = ((int)k * W + wave) * MARK, len = max(0, min(MARK, s.T - t0));
    rows<E, V, MARK, true, false> r;
    r.load(s, c, t0, s.T, x, gate, nullptr, starts);
    float m[MARK][V];
    uint32_t begin = r.begins(c);
    factor A[V]; float B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) B[v] = 0.0f;
#pragma unroll
    for (int t = 0; t < MARK; ++t) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            m[t][v] = t < len ? gate_of(get<E, V>(r.g[t], v)) : 0.0f;          // (behind the end: an open gate, h stays as it is)
            B[v] = step_of<E>(m[t][v], get<E, V>(r.x[t], v), (begin >> t) & 1 ? 0.0f : B[v]);
            A[v].step(m[t][v]);
        }
        pause<V>(t);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) { la[wave][v * 64 + lane] = A[v].held(begin != 0); lb[wave][v * 64 + lane] = B[v]; }
    forget<V>(m, begin); r.forget();
    __syncthreads();
    if constexpr (CHAIN) {
        __shared__ float lc[W][64 * V], ld[W][64 * V];
        pass_on<V, false, wide<E>>(ch, (int)k, s.chunks, plane, corner + floats / 4, c.valid, wave, lane, la, lb, lc, ld, carry);
    }
    float in[V], next[V];
    join<V, false, wide<E>>(la, lb, lane, W, wave, carry, in, next);
    if constexpr (CHAIN) leave<V, false>(ch, (int)k, s.chunks, plane, corner + floats / 4, c.valid, wave, next);
    if (marks && c.valid && len > 0) store_floats<V>(marks + (int64_t)(t0 / MARK) * plane + corner, floats, in);
    E* ph = h + (int64_t)t0 * plane + corner;
#pragma unroll
    for (int t = 0; t < MARK; ++t) {
        if (t < len) {
            vec o;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                in[v] = step_of<E>(m[t][v], get<E, V>(r.x[t], v), (begin >> t) & 1 ? 0.0f : in[v]);
                put<E, V>(o, v, in[v]);
            }
            if (c.valid) store_at<vec>(ph, elems, o);
            ph += plane;
        }
    }
    if (state_out && c.valid && len > 0 && t0 + len == s.T) store_floats<V>(state_out + corner, floats, in);          // (what h[T-1] was rounded from, not a join of maps)
}

// ---- gradients of a run.  hs: the states before each step, recomputed from the saved one --------------------------------------------------
template <typename E, int V> struct run_back {
    typedef vec_t<E, V> vec;
    rows<E, V, MARK, true, true> r;
    float h0[V];
    __device__ __forceinline__ void load(const shape& s, const columns<V>& c, int t0, int last, const E* x, const E* gate, const E* grad_h, const uint8_t* starts, const float* marks, int64_t plane, int64_t corner, uint32_t floats) {
        r.load(s, c, t0, last, x, gate, grad_h, starts);
        load_floats<V>(h0, marks + (int64_t)(min(t0, last - 1) / MARK) * plane + corner, floats);
    }
    __device__ __forceinline__ uint32_t states(const columns<V>& c, int len, float (&m)[MARK][V], float (&hs)[MARK][V]) {
        uint32_t begin = r.begins(c);
#pragma unroll
        for (int t = 0; t < MARK; ++t) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m[t][v] = t < len ? gate_of(get<E, V>(r.g[t], v)) : 0.0f;
                hs[t][v] = (begin >> t) & 1 ? 0.0f : h0[v];
                h0[v] = step_of<E>(m[t][v], get<E, V>(r.x[t], v), hs[t][v]);
            }
            pause<V>(t);
        }
        forget<V>(m, begin); r.forget();
        return begin;
    }
    // in: the gradient that arrives from behind the run, and then the one that leaves in front of it
    __device__ __forceinline__ void finish(const columns<V>& c, int t0, int len, uint32_t begin, const float (&m)[MARK][V], const float (&hs)[MARK][V], float (&in)[V], E* dx, E* dgate, int64_t plane, int64_t corner, uint32_t elems) {
        dx += (int64_t)(t0 + len - 1) * plane + corner;
        dgate += (int64_t)(t0 + len - 1) * plane + corner;
#pragma unroll
        for (int t = MARK - 1; t >= 0; --t) {
            if (t < len) {
                vec ox, og;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float l = get<E, V>(r.d[t], v) + in[v];
                    const float q = fabsf(m[t][v]), w = q * l, o = l - w;          // the smaller and the larger share
                    put<E, V>(ox, v, keeps(m[t][v]) ? w : o);
                    put<E, V>(og, v, times_apart<E>(fmaf(q, w, -w), get<E, V>(r.x[t], v), hs[t][v], 0.0f));
                    in[v] = (begin >> t) & 1 ? 0.0f : keeps(m[t][v]) ? o : w;
                }
                if (c.valid) { store_at<vec>(dx, elems, ox); store_at<vec>(dgate, elems, og); }
                dx -= plane; dgate -= plane;
            }
            pause<V>(MARK - 1 - t);
        }
    }
};

// whole: a wave runs back through all steps, a run ahead with its loads.  512 x 4096 x 128 bf16: 2.75 GB in 600 us, 4.6 TB/s; bound by memory.
template <typename E, int V>
__global__ __launch_bounds__(64) void k_memory_run_back(shape s, const E* __restrict__ x, const E* __restrict__ gate, const uint8_t* __restrict__ starts, const float* __restrict__ marks,
                                                            const E* __restrict__ grad_h, const float* __restrict__ grad_state, E* __restrict__ dx, E* __restrict__ dgate, float* __restrict__ dstate) {
    const columns<V> c(s.N, s.D);
    const int64_t plane = s.N * s.D, corner = c.n0 * s.D;
    const uint32_t elems = c.template bytes<E>(s.D), floats = c.template bytes<float>(s.D);
    float in[V];
#pragma unroll
    for (int v = 0; v < V; ++v) in[v] = 0.0f;
    if (grad_state) load_floats<V>(in, grad_state + corner, floats);
    auto load = [&](run_back<E, V>& b, int t0) { b.load(s, c, max(t0, 0), s.T, x, gate, grad_h, starts, marks, plane, corner, floats); };          // (in front of the first run: that again)
    auto one = [&](run_back<E, V>& b, int t0) {
        const int len = min(MARK, s.T - t0);
        float m[MARK][V], hs[MARK][V];
        const uint32_t begin = b.states(c, len, m, hs);
        b.finish(c, t0, len, begin, m, hs, in, dx, dgate, plane, corner, elems);
    };
    run_back<E, V> p, q;
    int t0 = (s.T - 1) / MARK * MARK;
    load(p, t0);
    for (;;) {
        load(q, t0 - MARK);
        one(p, t0);
        if ((t0 -= MARK) < 0) break;
        load(p, t0 - MARK);
        one(q, t0);
        if ((t0 -= MARK) < 0) break;
    }
    if (dstate && c.valid) store_floats<V>(dstate + corner, floats, in);
}

// short and chain, back: 128 x 128 x 512 bf16: 86 MB in 28.8 us, 3.0 TB/s, two waves per SIMD unit with a run each, vector units 0.50 busy; 2048 x 8 x 512 float32: 170 MB in 40 us, 4.2 TB/s.
template <typename E, int V, int W, bool CHAIN>
__global__ __launch_bounds__(64 * W) void k_memory_short_back(shape s, chain ch, const E* __restrict__ x, const E* __restrict__ gate, const uint8_t* __restrict__ starts, const float* __restrict__ marks,
                                                              const E* __restrict__ grad_h, const float* __restrict__ grad_state, E* __restrict__ dx, E* __restrict__ dgate, float* __restrict__ dstate) {
    __shared__ float la[W][64 * V], lb[W][64 * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t place = CHAIN ? take_ticket(ch) : blockIdx.x, back = CHAIN ? place / ch.blocks : 0;
    const columns<V> c(s.N, s.D, CHAIN ? place - back * ch.blocks : place);
    const int k = CHAIN ? s.chunks - 1 - (int)back : 0;
    const int64_t plane = s.N * s.D, corner = c.n0 * s.D;
    const uint32_t elems = c.template bytes<E>(s.D), floats = c.template bytes<float>(s.D);
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = 0.0f;
    if (grad_state) load_floats<V>(carry, grad_state + corner, floats);
    const int t0 = (k * W + wave) * MARK, len = max(0, min(MARK, s.T - t0));
    run_back<E, V> b;
    b.load(s, c, t0, s.T, x, gate, grad_h, starts, marks, plane, corner, floats);
    float m[MARK][V], hs[MARK][V];
    uint32_t begin = b.states(c, len, m, hs);
    factor A[V]; float B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) B[v] = 0.0f;
#pragma unroll
    for (int t = MARK - 1; t >= 0; --t) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            B[v] = (begin >> t) & 1 ? 0.0f : decay_of(m[t][v], (t < len ? get<E, V>(b.r.d[t], v) : 0.0f) + B[v]);
            A[v].step(m[t][v]);
        }
        pause<V>(MARK - 1 - t);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) { la[wave][v * 64 + lane] = A[v].held(begin != 0); lb[wave][v * 64 + lane] = B[v]; }
    forget<V>(m, begin); b.r.forget();
    __syncthreads();
    if constexpr (CHAIN) {
        __shared__ float lc[W][64 * V], ld[W][64 * V];
        pass_on<V, true, false>(ch, k, s.chunks, plane, corner + floats / 4, c.valid, wave, lane, la, lb, lc, ld, carry);
    }
    float in[V], next[V];
    join<V, true, false>(la, lb, lane, W, W - 1 - wave, carry, in, next);
    if constexpr (CHAIN) leave<V, true>(ch, k, s.chunks, plane, corner + floats / 4, c.valid, wave, next);
    if (len > 0) b.finish(c, t0, len, begin, m, hs, in, dx, dgate, plane, corner, elems);
    if (dstate && wave == 0 && c.valid && k == 0) store_floats<V>(dstate + corner, floats, in);
}

// One control step.  state_out may be state: a thread reads its own columns, which are no other's, before it writes them.
// 8 x 512 float32: 2.6 to 2.8 us, a launch; 4096 x 512 bf16: 29 MB in 5.0 to 5.3 us, 5.5 TB/s and more from the last-level cache.
template <typename E, int V>
__global__ __launch_bounds__(256) void k_memory_step(int64_t N, int64_t D, int64_t x_n, int64_t gate_n, int64_t starts_n, const E* __restrict__ x, const E* __restrict__ gate,
                                                     const uint8_t* __restrict__ starts, const float* state, E* __restrict__ h, float* state_out) {
    typedef vec_t<E, V> vec;
    const int64_t per = D / V, q = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (q >= N * per) return;
    const int64_t n = q / per, d = (q - n * per) * V, col = n * D + d;
    const vec xs = *(const vec*)(x + n * x_n + d), gs = *(const vec*)(gate + n * gate_n + d);
    const bool begin = starts && starts[n * starts_n];
    vec o;
    vec_t<float, V> last;
    float r[V];
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = 0.0f;
    if (state) {
        const vec_t<float, V> f = *(const vec_t<float, V>*)(state + col);
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = get<float, V>(f, v);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        r[v] = step_of<E>(gate_of(get<E, V>(gs, v)), get<E, V>(xs, v), begin ? 0.0f : r[v]);
        put<E, V>(o, v, r[v]);
        put<float, V>(last, v, r[v]);
    }
    *(vec*)(h + col) = o;
    *(vec_t<float, V>*)(state_out + col) = last;
}

}  // namespace dlm
