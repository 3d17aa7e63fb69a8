// dl_memory.hpp -- the gated memory of a recurrent policy over a rollout: forward, gradients, one control step.
//
//     a = sigmoid(g), s = 1 - a:      h[t] = a h' + s x[t],   h' = start ? 0 : h[t-1]
//     l[t] = dh[t] + c[t+1],  c[t] = start ? 0 : a l[t]:      dx = s l,   dg = (h' - x) a s l,   dstate = c[0]
//
// Bound by memory: three elements moved per step forward, five backward.  Every element is loaded once: a wave keeps MARK steps
// of 64 columns in registers, reduces them to the affine map (A, B) of its run, the waves of a workgroup exchange their maps
// through LDS, and each wave then finishes its own steps from the registers.  With too few columns for the chip the time axis is
// also cut into chunks over workgroups: a first kernel reduces every chunk to its map, the second starts from the maps before it.
//
// Rounding.  The smaller of a and s is computed as e / (1 + e), e = exp(-|g|), and both products go through it:
//     g >= 0:  h = h' + s (x - h'),  c = l - s l        g < 0:  h = x + a (h' - x),  c = a l
// so that a long memory (s small) loses nothing to the rounding of a = 1 - s, and a closed gate gives x exactly.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dlm {

constexpr int MARK = 16;          // steps of a wave's run, and between two saved states

template <typename E, int V> struct vec { typedef E type __attribute__((ext_vector_type(V))); };
template <typename E> struct vec<E, 1> { typedef E type; };
template <typename E, int V> using vec_t = typename vec<E, V>::type;

template <typename E, int V> __device__ __forceinline__ float get(const vec_t<E, V>& v, int i) {
    if constexpr (V == 1) return (float)v; else return (float)v[i];
}
template <typename E, int V> __device__ __forceinline__ void put(vec_t<E, V>& v, int i, float f) {
    if constexpr (V == 1) v = (E)f; else v[i] = (E)f;
}

struct shape {
    int64_t T, N, D;
    int64_t x_t, x_n, gate_t, gate_n, starts_t, starts_n, grad_t, grad_n;
    int64_t chunk;                // steps of a workgroup (a multiple of waves * MARK)
    int32_t chunks;
};

// min(a, s), with the sign of the gate: >= +0 where a is the larger one (g >= 0), <= -0 where s is.
// exp(-|g|) with the rounding of |g| log2(e) carried along: one unit of the result, far tails included.
__device__ __forceinline__ float gate_of(float g) {
    const float u = -fabsf(g);
    const float p = u * 1.44269504f;
    const float r = fmaf(u, 1.44269504f, -p) + u * 1.92596299e-8f;
    float e = __builtin_amdgcn_exp2f(p);
    e = fmaf(e, r * 0.693147181f, e);
    if (p < -150.0f) e = 0.0f;                         // (infinite gates: r is NaN)
    const float m = e * __builtin_amdgcn_rcpf(1.0f + e);
    return g >= 0.0f ? m : (g < 0.0f ? -m : g);        // a NaN stays one
}
__device__ __forceinline__ bool keeps(float m) { return !(__float_as_uint(m) >> 31); }
// Between the passes over a run: the comparisons of the first are made again instead of being kept, a pair of scalar registers each.
template <int V> __device__ __forceinline__ void forget(float (&m)[MARK][V], uint32_t& begin) {
#pragma unroll
    for (int t = 0; t < MARK; ++t) {
#pragma unroll
        for (int v = 0; v < V; ++v) asm volatile("" : "+v"(m[t][v]));
    }
    asm volatile("" : "+v"(begin));
}
// one step of the state
__device__ __forceinline__ float step_of(float m, float x, float h) {
    const float d = x - h;
    return keeps(m) ? fmaf(m, d, h) : fmaf(m, d, x);   // (m < 0: x + |m| (h - x) = x + m (x - h))
}
// one step of a product of a
__device__ __forceinline__ float decay_of(float m, float l) { return keeps(m) ? fmaf(-m, l, l) : -m * l; }

// The map h -> a h + b of a run, a = the product of its steps'.  Like a step it is held by the smaller of a and p = 1 - a: m = p
// where p <= 1/2, else -a; so a product over thousands of open gates is as exact as its steps.  BEGUN: an episode began inside
// the run, nothing before it counts, not even a NaN.
constexpr float BEGUN = 2.0f;
struct factor {
    float a = 1.0f, p = 0.0f;
    __device__ __forceinline__ void step(float m) {
        p = fmaf(keeps(m) ? m : 1.0f + m, a, p);
        a = decay_of(m, a);
    }
    __device__ __forceinline__ float held(bool begun) const { return begun ? BEGUN : p <= 0.5f ? p : -a; }          // (a NaN stays one)
};
__device__ __forceinline__ float apply(float m, float b, float h) { return m > 1.0f ? b : decay_of(m, h) + b; }
__device__ __forceinline__ float after(float m, float n) {          // m, then n
    if (m > 1.0f || n > 1.0f) return BEGUN;
    factor f;
    f.step(m); f.step(n);
    return f.held(false);
}

template <int V> struct columns {
    int64_t n, d, col;            // walker, channel, place in an [N, D] array
    bool valid;
    __device__ columns(int64_t N, int64_t D) {
        const int64_t per = D / V;
        const int64_t q = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
        valid = q < N * per;
        n = valid ? q / per : 0;
        d = valid ? (q - n * per) * V : 0;
        col = n * D + d;
    }
};

// The state (or gradient) that enters the run of each wave from the maps of the waves before it, and the one behind the last.
// `from` = how many maps come first in the order of the recurrence for this wave.
template <int V>
__device__ __forceinline__ void join(const float (*la)[64 * V], const float (*lb)[64 * V], int lane, int waves, int from, const float (&carry)[V], float (&mine)[V], float (&next)[V], bool back) {
#pragma unroll
    for (int v = 0; v < V; ++v) next[v] = mine[v] = carry[v];
    for (int i = 0; i < waves; ++i) {
        const int w = back ? waves - 1 - i : i;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            next[v] = apply(la[w][v * 64 + lane], lb[w][v * 64 + lane], next[v]);
            if (i + 1 == from) mine[v] = next[v];
        }
    }
}

// Maps of whole chunks -> the value that enters chunk k, by the whole workgroup: every wave joins a part of the chunks before.
// maps: float [chunks][2][N * D].
template <int V, bool BACK>
__device__ __forceinline__ void enter(const float* maps, int64_t plane, int k, int chunks, const columns<V>& c, int waves, int wave, int lane, float (*la)[64 * V], float (*lb)[64 * V], float (&carry)[V]) {
    const int before = BACK ? chunks - 1 - k : k;
    if (before == 0) return;
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 0.0f; B[v] = 0.0f; }
    const int lo = (int)((int64_t)before * wave / waves), hi = (int)((int64_t)before * (wave + 1) / waves);
#pragma unroll 4
    for (int i = lo; i < hi; ++i) {
        const int j = BACK ? chunks - 1 - i : i;
        const float* p = maps + (int64_t)j * 2 * plane + c.col;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float a = p[v], b = p[plane + v];
            B[v] = apply(a, b, B[v]);
            A[v] = after(A[v], a);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) { la[wave][v * 64 + lane] = A[v]; lb[wave][v * 64 + lane] = B[v]; }
    __syncthreads();
    float mine[V], next[V];
    join<V>(la, lb, lane, waves, 0, carry, mine, next, false);
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = next[v];
    __syncthreads();
}

// MAPS: only reduce the chunk to its map.
template <typename E, int V, int W, bool MAPS>
__global__ __launch_bounds__(64 * W) void k_memory_forward(shape s, const E* __restrict__ x, const E* __restrict__ gate, const uint8_t* __restrict__ starts, const float* __restrict__ state,
                                                           E* __restrict__ h, float* __restrict__ state_out, float* __restrict__ marks, float* __restrict__ maps) {
    typedef vec_t<E, V> vec;
    __shared__ float la[W][64 * V], lb[W][64 * V];
    const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const columns<V> c(s.N, s.D);
    const int64_t plane = s.N * s.D;
    const int k = blockIdx.y;
    const int64_t first = (int64_t)k * s.chunk, last = min(first + s.chunk, s.T);
    float carry[V], chunk[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { carry[v] = 0.0f; chunk[v] = 0.0f; }
    if (!MAPS) {
        if (state) {
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = state[c.col + v];
        }
        if (s.chunks > 1) enter<V, false>(maps, plane, k, s.chunks, c, W, wave, lane, la, lb, carry);
    }
    for (int64_t base = first; base < last; base += W * MARK) {
        const int64_t t0 = base + wave * MARK;
        const int len = (int)max((int64_t)0, min((int64_t)MARK, last - t0));
        // Rows behind the end read the last one again and count as steps with an open gate (h stays as it is).
        vec xs[MARK], gs[MARK]; float m[MARK][V]; uint8_t bs[MARK]; uint32_t begin = 0;
#pragma unroll
        for (int t = 0; t < MARK; ++t) {
            const int64_t row = min(t0 + t, last - 1);
            xs[t] = *(const vec*)(x + row * s.x_t + c.n * s.x_n + c.d);
            gs[t] = *(const vec*)(gate + row * s.gate_t + c.n * s.gate_n + c.d);
            bs[t] = starts ? starts[row * s.starts_t + c.n * s.starts_n] : 0;
        }
#pragma unroll
        for (int t = 0; t < MARK; ++t) {
#pragma unroll
            for (int v = 0; v < V; ++v) m[t][v] = t < len ? gate_of(get<E, V>(gs[t], v)) : 0.0f;
            if (t < len && bs[t]) begin |= 1u << t;
        }
        float in[V];
        if (W > 1 || MAPS) {
            factor A[V]; float B[V];
#pragma unroll
            for (int v = 0; v < V; ++v) B[v] = 0.0f;
#pragma unroll
            for (int t = 0; t < MARK; ++t) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    B[v] = step_of(m[t][v], get<E, V>(xs[t], v), (begin >> t) & 1 ? 0.0f : B[v]);
                    A[v].step(m[t][v]);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) { la[wave][v * 64 + lane] = A[v].held(begin != 0); lb[wave][v * 64 + lane] = B[v]; }
            forget<V>(m, begin);
            __syncthreads();
            float next[V];
            join<V>(la, lb, lane, W, wave, carry, in, next, false);
            if (MAPS) {
                for (int w = 0; w < W; ++w) {
#pragma unroll
                    for (int v = 0; v < V; ++v) chunk[v] = after(chunk[v], la[w][v * 64 + lane]);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = next[v];
            __syncthreads();
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) in[v] = carry[v];
        }
        if (!MAPS) {
            if (marks && c.valid && len > 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) marks[(t0 / MARK) * plane + c.col + v] = in[v];
            }
            E* ph = h + t0 * plane + c.col;
#pragma unroll
            for (int t = 0; t < MARK; ++t) {
                if (t < len) {
                    vec o;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        in[v] = step_of(m[t][v], get<E, V>(xs[t], v), (begin >> t) & 1 ? 0.0f : in[v]);
                        put<E, V>(o, v, in[v]);
                    }
                    if (c.valid) *(vec*)(ph + t * plane) = o;
                }
            }
            if (W == 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) carry[v] = in[v];
            }
        }
    }
    if (MAPS) {
        if (wave == 0 && c.valid) {
            float* p = maps + (int64_t)k * 2 * plane + c.col;
#pragma unroll
            for (int v = 0; v < V; ++v) { p[v] = chunk[v]; p[plane + v] = carry[v]; }
        }
    } else if (state_out && wave == 0 && c.valid && last == s.T) {
#pragma unroll
        for (int v = 0; v < V; ++v) state_out[c.col + v] = carry[v];
    }
}

template <typename E, int V, int W, bool MAPS>
__global__ __launch_bounds__(64 * W) void k_memory_backward(shape s, const E* __restrict__ x, const E* __restrict__ gate, const uint8_t* __restrict__ starts, const float* __restrict__ marks,
                                                            const E* __restrict__ grad_h, const float* __restrict__ grad_state, E* __restrict__ dx, E* __restrict__ dgate,
                                                            float* __restrict__ dstate, float* __restrict__ maps) {
    typedef vec_t<E, V> vec;
    __shared__ float la[W][64 * V], lb[W][64 * V];
    const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const columns<V> c(s.N, s.D);
    const int64_t plane = s.N * s.D;
    const int k = blockIdx.y;
    const int64_t first = (int64_t)k * s.chunk, last = min(first + s.chunk, s.T);
    float carry[V], chunk[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { carry[v] = 0.0f; chunk[v] = 0.0f; }
    if (!MAPS) {
        if (grad_state) {
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = grad_state[c.col + v];
        }
        if (s.chunks > 1) enter<V, true>(maps, plane, k, s.chunks, c, W, wave, lane, la, lb, carry);
    }
    const int64_t span = W * MARK;
    for (int64_t base = first + (last - first - 1) / span * span; base >= first; base -= span) {
        const int64_t t0 = base + wave * MARK;
        const int len = (int)max((int64_t)0, min((int64_t)MARK, last - t0));
        vec xs[MARK], gs[MARK], ds[MARK]; float m[MARK][V], hs[MARK][V], h0[V]; uint8_t bs[MARK]; uint32_t begin = 0;
        if (!MAPS) {
            const int64_t mark = min(t0, last - 1) / MARK;
#pragma unroll
            for (int v = 0; v < V; ++v) h0[v] = marks[mark * plane + c.col + v];
        }
#pragma unroll
        for (int t = 0; t < MARK; ++t) {
            const int64_t row = min(t0 + t, last - 1);
            if (!MAPS) xs[t] = *(const vec*)(x + row * s.x_t + c.n * s.x_n + c.d);
            gs[t] = *(const vec*)(gate + row * s.gate_t + c.n * s.gate_n + c.d);
            if (grad_h && t < len) ds[t] = *(const vec*)(grad_h + row * s.grad_t + c.n * s.grad_n + c.d);
            else {
#pragma unroll
                for (int v = 0; v < V; ++v) put<E, V>(ds[t], v, 0.0f);
            }
            bs[t] = starts ? starts[row * s.starts_t + c.n * s.starts_n] : 0;
        }
#pragma unroll
        for (int t = 0; t < MARK; ++t) {
            if (t < len && bs[t]) begin |= 1u << t;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m[t][v] = t < len ? gate_of(get<E, V>(gs[t], v)) : 0.0f;
                if (!MAPS) {
                    hs[t][v] = (begin >> t) & 1 ? 0.0f : h0[v];
                    h0[v] = step_of(m[t][v], get<E, V>(xs[t], v), hs[t][v]);
                }
            }
        }
        forget<V>(m, begin);
        float in[V];
        if (W > 1 || MAPS) {
            factor A[V]; float B[V];
#pragma unroll
            for (int v = 0; v < V; ++v) B[v] = 0.0f;
#pragma unroll
            for (int t = MARK - 1; t >= 0; --t) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    B[v] = (begin >> t) & 1 ? 0.0f : decay_of(m[t][v], get<E, V>(ds[t], v) + B[v]);
                    A[v].step(m[t][v]);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) { la[wave][v * 64 + lane] = A[v].held(begin != 0); lb[wave][v * 64 + lane] = B[v]; }
            forget<V>(m, begin);
            __syncthreads();
            float next[V];
            join<V>(la, lb, lane, W, W - 1 - wave, carry, in, next, true);
            if (MAPS) {
                for (int w = 0; w < W; ++w) {
#pragma unroll
                    for (int v = 0; v < V; ++v) chunk[v] = after(chunk[v], la[w][v * 64 + lane]);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = next[v];
            __syncthreads();
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) in[v] = carry[v];
        }
        if (!MAPS) {
            E* pdx = dx + t0 * plane + c.col;
            E* pdg = dgate + t0 * plane + c.col;
#pragma unroll
            for (int t = MARK - 1; t >= 0; --t) {
                if (t < len) {
                    vec ox, og;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const float q = fabsf(m[t][v]), l = get<E, V>(ds[t], v) + in[v];
                        const float s_ = keeps(m[t][v]) ? q : 1.0f - q;
                        put<E, V>(ox, v, s_ * l);
                        put<E, V>(og, v, (hs[t][v] - get<E, V>(xs[t], v)) * ((q - q * q) * l));
                        in[v] = (begin >> t) & 1 ? 0.0f : decay_of(m[t][v], l);
                    }
                    if (c.valid) { *(vec*)(pdx + t * plane) = ox; *(vec*)(pdg + t * plane) = og; }
                }
            }
            if (W == 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) carry[v] = in[v];
            }
        }
    }
    if (MAPS) {
        if (wave == 0 && c.valid) {
            float* p = maps + (int64_t)k * 2 * plane + c.col;
#pragma unroll
            for (int v = 0; v < V; ++v) { p[v] = chunk[v]; p[plane + v] = carry[v]; }
        }
    } else if (dstate && wave == 0 && c.valid && first == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) dstate[c.col + v] = carry[v];
    }
}

// One control step.  state_out may be state: a thread reads its own columns before it writes them.
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
    float r[V];
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = state && !begin ? state[col + v] : 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        r[v] = step_of(gate_of(get<E, V>(gs, v)), get<E, V>(xs, v), r[v]);
        put<E, V>(o, v, r[v]);
    }
    *(vec*)(h + col) = o;
#pragma unroll
    for (int v = 0; v < V; ++v) state_out[col + v] = r[v];
}

}  // namespace dlm
