// dl_orth.hpp -- orthogonalisation of an update by Newton-Schulz products, and the weight update built on it.
//
//     X = G / |G|_F (from the short side: X is [m, n], m <= n);  repeat:  A = X X',  Q = a I + b A + c A A,  X = Q X
//
// Bound by the matrix cores.  A product of 32-bit matrices on them would run at a sixteenth of the 16-bit rate, and one rounding of X
// to 16 bits is amplified by up to a^steps (485 for five steps) in the directions of small singular values.  So every matrix is
// held as the sum of two float16 planes, hi + lo = 22 bits, and a product is three 16-bit ones accumulated in 32 bits,
// hi hi + hi lo + lo hi (what is left out is below 2^-22): the splitting of Ootomo and Yokota (2022).  All entries are at most
// about one, so they are held times 2^10, which keeps lo clear of float16's smallest numbers.
// That goes for every step and every type of result: a result of 16 bits is the 32-bit one, rounded once.
// A and Q are symmetric: only their tiles on and below the diagonal are computed, and written to both places.
//
// Layout.  A matrix that is an operand lies in memory as the matrix cores read it: for 16 rows and 32 columns k a "fragment" of
// [plane][lane][8] float16, lane = row + 16 * (k / 8), 2 KB; fragments of a row block follow each other along k.  Copies to LDS and
// reads from it are then straight runs of 16 bytes per lane without bank conflicts, and every product has the form
// C[i][j] = sum_k P[i][k] Q[j][k].  X is kept in both orientations (XR: rows i, XC: rows j) because A needs one and Q X the other.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dlo {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4_ __attribute__((ext_vector_type(4)));

constexpr float SCALE = 1024.0f;
constexpr int FRAG = 1024;            // float16 of a fragment: two planes of 64 lanes x 8

// Where a matrix [batch][rows][cols] of the caller lies, seen from the short side: element (i, j), i < m, j < n, at i * si + j * sj.
struct matrix {
    int64_t b, si, sj;
};

struct plan {
    int32_t m, n, mp, np;             // short and long side, and what they are padded to
    int64_t x_size, a_size;           // float16 of one X, one A
    int32_t partials;
};

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

template <typename E> __device__ __forceinline__ float load_as(const void* p, int64_t i) { return (float)((const E*)p)[i]; }
__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
    return dtype == 0 ? load_as<float>(p, i) : dtype == 1 ? load_as<__bf16>(p, i) : load_as<_Float16>(p, i);
}
__device__ __forceinline__ void store_elem(void* p, int dtype, int64_t i, float v) {
    if (dtype == 0) ((float*)p)[i] = v;
    else if (dtype == 1) ((__bf16*)p)[i] = (__bf16)v;
    else ((_Float16*)p)[i] = (_Float16)v;
}

// four neighbours, at any alignment
template <typename E> __device__ __forceinline__ float4_ load4_as(const void* p, int64_t i) {
    typedef E vec __attribute__((ext_vector_type(4), aligned(sizeof(E))));
    const vec v = *(const vec*)((const E*)p + i);
    return float4_{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
__device__ __forceinline__ float4_ load4(const void* p, int dtype, int64_t i) {
    return dtype == 0 ? load4_as<float>(p, i) : dtype == 1 ? load4_as<__bf16>(p, i) : load4_as<_Float16>(p, i);
}
template <typename E> __device__ __forceinline__ void store4_as(void* p, int64_t i, float4_ v) {
    typedef E vec __attribute__((ext_vector_type(4), aligned(sizeof(E))));
    *(vec*)((E*)p + i) = vec{(E)v[0], (E)v[1], (E)v[2], (E)v[3]};
}
__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, float4_ v) {
    if (dtype == 0) store4_as<float>(p, i, v);
    else if (dtype == 1) store4_as<__bf16>(p, i, v);
    else store4_as<_Float16>(p, i, v);
}

// ---- the sum of squares, in 64 bits (a float32 gradient of 1e30 or of 1e-30 is as good as another) --------------------------------
// With a momentum: m' = beta m + g first, and the matrix is g + beta m' (nesterov) or m'.  rows x cols as the caller sees them.
struct source {
    const void* g; int dtype;
    const float* m; float* m_out;     // NULL: no momentum
    float beta; int nesterov;
    int64_t g_b, g_r, m_b, m_r, o_b, o_r;          // strides of g, m, m_out: matrix, row
};

// Four neighbours of a row (`n` of them, where fewer are left): everything is loaded, for several places at once, before the first is used.
struct place {
    int64_t b, r, c;
    int n;
    float4_ u, v;          // gradient and momentum, then what the update is made of
    __device__ __forceinline__ void load(const source& s, bool first) {
        u = v = float4_{};
        const int64_t g = b * s.g_b + r * s.g_r + c;
        if (n >= 4) u = load4(s.g, s.dtype, g);
        else for (int e = 0; e < n; ++e) u[e] = load_elem(s.g, s.dtype, g + e);
        if (s.m && n > 0) {
            const float* m = first ? s.m + b * s.m_b + r * s.m_r + c : s.m_out + b * s.o_b + r * s.o_r + c;
            if (n >= 4) v = load4_as<float>(m, 0);
            else for (int e = 0; e < n; ++e) v[e] = m[e];
        }
    }
    __device__ __forceinline__ void move(const source& s, bool first) {
        if (!s.m || n <= 0) return;
        if (first) {
            for (int e = 0; e < 4; ++e) v[e] = fmaf(s.beta, v[e], u[e]);
            float* o = s.m_out + b * s.o_b + r * s.o_r + c;
            if (n >= 4) store4_as<float>(o, 0, v);
            else for (int e = 0; e < n; ++e) o[e] = v[e];
        }
        for (int e = 0; e < 4; ++e) u[e] = s.nesterov ? fmaf(s.beta, v[e], u[e]) : v[e];
    }
};

// rows x cols as they are read: one long row where the rows of all arrays follow each other
// (and counters for later kernels to zero).  4096 x 8192 bf16: 67 MB in 32 us, 2.1 TB/s, half of what memory gives; 0.5 % of the update.
__global__ __launch_bounds__(256) void k_orth_norm(source s, int64_t rows, int64_t cols, double* __restrict__ partials, uint32_t* __restrict__ counters, int n_counters) {
    if (blockIdx.x == 0 && blockIdx.y == 0) for (int k = threadIdx.x; k < n_counters; k += 256) counters[k] = 0;
    constexpr int AT_ONCE = 4;
    const int64_t per = (cols + 3) / 4, all = rows * per, step = (int64_t)gridDim.x * 256;          // in fours
    double sum = 0.0;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < all; e += AT_ONCE * step) {
        place p[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int64_t f = e + k * step, r = rows == 1 ? 0 : f / per;
            p[k].b = blockIdx.y; p[k].r = r; p[k].c = (f - r * per) * 4;
            p[k].n = f < all ? (int)min((int64_t)4, cols - p[k].c) : 0;
            p[k].load(s, true);
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            p[k].move(s, true);
            for (int q = 0; q < 4; ++q) sum += (double)p[k].u[q] * p[k].u[q];
        }
    }
    __shared__ double part[4];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partials[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// ---- X = G / |G| into both orientations: one workgroup per 64 x 64 ---------------------------------------------------------------
// 4096 x 8192 bf16: 335 MB in 76 to 81 us, 4.1 to 4.4 TB/s; bound by memory.
__global__ __launch_bounds__(256) void k_orth_load(source s, plan p, int turned, const double* __restrict__ partials, _Float16* __restrict__ xr, _Float16* __restrict__ xc) {
    const int b = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float tile[64][65];          // [short side][long side]
    const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    const int r0 = turned ? j0 : i0, c0 = turned ? i0 : j0, rows = turned ? p.n : p.m, cols = turned ? p.m : p.n;
    place at[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        at[e].b = b; at[e].r = r0 + e * 16 + (threadIdx.x >> 4); at[e].c = c0 + (threadIdx.x & 15) * 4;
        at[e].n = at[e].r < rows ? min(4, cols - (int)at[e].c) : 0;
        at[e].load(s, false);
    }
    double sum = 0.0;
    for (int k = lane; k < p.partials; k += 64) sum += partials[(int64_t)b * p.partials + k];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    const double inv = sum != 0.0 ? (double)SCALE / sqrt(sum) : 0.0;          // (NaN != 0)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        at[e].move(s, false);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = e * 16 + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 4 + k;
            (turned ? tile[c][r] : tile[r][c]) = (float)(at[e].u[k] * inv);
        }
    }
    __syncthreads();
    // 4 x 2 fragments with rows i and 4 x 2 with rows j
#pragma unroll
    for (int f = wave; f < 16; f += 4) {
        const bool c_side = f >= 8;
        const int row = (f & 3) * 16 + (lane & 15), k = (f >> 2 & 1) * 32 + (lane >> 4) * 8;
        const int first = c_side ? j0 : i0, second = c_side ? i0 : j0, rows_ = c_side ? p.np : p.mp, ks = c_side ? p.mp : p.np;
        if (first + (f & 3) * 16 >= rows_ || second + (f >> 2 & 1) * 32 >= ks) continue;
        half8 hi, lo;
#pragma unroll
        for (int q = 0; q < 8; ++q) { _Float16 h, l; split(c_side ? tile[k + q][row] : tile[row][k + q], h, l); hi[q] = h; lo[q] = l; }
        const int64_t block = first / 16 + (f & 3), kb = second / 32 + (f >> 2 & 1);
        _Float16* to = (c_side ? xc : xr) + b * p.x_size + (block * (ks / 32) + kb) * FRAG + lane * 8;
        *(half8*)to = hi;
        *(half8*)(to + 512) = lo;
    }
}

// ---- the products ----------------------------------------------------------------------------------------------------------------
enum { GRAM, POLY, STEP, LAST };      // A = XR XR';  Q = aI + bA + cAA;  X = Q X as the next operand;  X = Q X as the result

struct product {
    const _Float16* P; const _Float16* Q;          // operands, [rows / 16][kb][FRAG]
    int64_t P_b, Q_b;
    int32_t kb;                                    // steps of 32 along k
    int32_t tiles_i, tiles_j, tiles, whole;        // tiles, and those of them that are not cut up
    _Float16* out0; int64_t out0_b, out0_kb;       // GRAM, POLY: the symmetric result;  STEP: XR
    _Float16* out1; int64_t out1_b, out1_kb;       // STEP: XC
    const _Float16* A;                             // POLY: as out0
    float a, b, c;
    // GRAM of k_orth_direct with `splits` workgroups per tile along k: their sums, and a counter per tile that is zero before and after
    int32_t splits;
    float* parts; uint32_t* arrived;
    // LAST: out = keep * w + gain * X
    void* out; const void* w; int out_type, w_type;
    matrix out_at, w_at;
    float keep, gain;
    int32_t m, n;
};

__device__ __forceinline__ void below(int t, int& ti, int& tj) {          // the tiles on and below the diagonal, row by row
    ti = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    while (ti * (ti + 1) / 2 > t) --ti;
    tj = t - ti * (ti + 1) / 2;
}

// out = keep w + gain X for the I x J values of `tile` (at [i * pitch + j]) from (i0, j0) on, in fours along the caller's rows
template <int I, int J, int THREADS>
__device__ __forceinline__ void emit(const product& p, int64_t b, const float* tile, int pitch, int i0, int j0) {
    const float gain = p.gain / (SCALE * SCALE);
    // the caller's rows run along the short side; along the long one if they have one element each, which follow each other in every array
    const bool down = p.out_at.si == 1 && (p.out_at.sj != 1 || (p.w && p.w_at.sj != 1));
#pragma unroll 4
    for (int e = threadIdx.x; e < I * J / 4; e += THREADS) {
        const int i = down ? e % (I / 4) * 4 : e / (J / 4), j = down ? e / (I / 4) : e % (J / 4) * 4;
        const int left = i0 + i < p.m && j0 + j < p.n ? down ? p.m - i0 - i : p.n - j0 - j : 0;
        const float* t = tile + i * pitch + j;
        const int d = down ? pitch : 1;
        float4_ v = {t[0] * gain, t[d] * gain, t[2 * d] * gain, t[3 * d] * gain};
        const int64_t at = b * p.out_at.b + (i0 + i) * p.out_at.si + (j0 + j) * p.out_at.sj, wat = b * p.w_at.b + (i0 + i) * p.w_at.si + (j0 + j) * p.w_at.sj;
        if (left >= 4) {
            if (p.w) {
                const float4_ w = load4(p.w, p.w_type, wat);
                for (int k = 0; k < 4; ++k) v[k] = fmaf(p.keep, w[k], v[k]);
            }
            store4(p.out, p.out_type, at, v);
        } else {
            for (int k = 0; k < left; ++k) store_elem(p.out, p.out_type, at + k, p.w ? fmaf(p.keep, load_elem(p.w, p.w_type, wat + k), v[k]) : v[k]);
        }
    }
}

template <bool V> struct flag { static constexpr bool value = V; };
template <int N> struct number { static constexpr int value = N; };

// A tile of BM x BN in waves of WM x WN, NS steps of operands in LDS.
template <int BM, int BN, int WM, int WN, int NS> struct staged {
    static constexpr int WAVES = (BM / WM) * (BN / WN), ROWS = BM / 16 + BN / 16;          // fragments of a step
    static constexpr int PITCH = BN + 4, STAGE = ROWS * FRAG * 2;                          // bytes
    static constexpr int BYTES = NS * STAGE > BM * PITCH * 4 ? NS * STAGE : BM * PITCH * 4;
    static constexpr int MOVES = ROWS * 2 / WAVES;                                         // copies of a wave and step
    static_assert(ROWS * 2 % WAVES == 0, "every wave moves the same number of pieces");
};

// The finished tile in LDS (BM x BN sums, [i * PITCH + j]) on its way to memory.
template <int BM, int BN, int WAVES, int MODE>
__device__ __forceinline__ void finish(const product& p, float* tile, int i0, int j0) {
    constexpr int PITCH = BN + 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t b = blockIdx.z;
    const int row = lane & 15, k8 = (lane >> 4) * 8;
    if (MODE == LAST) {
        emit<BM, BN, WAVES * 64>(p, b, tile, PITCH, i0, j0);
        return;
    }
    // rows i, k along j.  Of a symmetric result only the blocks of 32 on and below the diagonal count.
    constexpr bool HALF = MODE == GRAM || MODE == POLY;
    for (int f = wave; f < (BM / 16) * (BN / 32); f += WAVES) {
        const int ri = f / (BN / 32), kj = f % (BN / 32);
        if (HALF && i0 / 32 + ri / 2 < j0 / 32 + kj) continue;
        const int64_t at = (((int64_t)(i0 / 16 + ri)) * p.out0_kb + j0 / 32 + kj) * FRAG + lane * 8;
        float* src = tile + (ri * 16 + row) * PITCH + kj * 32 + k8;
        half8 hi, lo, ah, al;
        if (MODE == POLY) { const _Float16* A = p.A + b * p.out0_b + at; ah = *(const half8*)A; al = *(const half8*)(A + 512); }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            float v = src[q] * (1.0f / SCALE);
            if (MODE == POLY) {
                v = fmaf(p.c, v, p.b * ((float)ah[q] + (float)al[q]));
                if (i0 + ri * 16 + row == j0 + kj * 32 + k8 + q) v += p.a * SCALE;
                src[q] = v * SCALE;           // for the other orientation
            }
            _Float16 h, l; split(v, h, l); hi[q] = h; lo[q] = l;
        }
        _Float16* to = p.out0 + b * p.out0_b + at;
        *(half8*)to = hi; *(half8*)(to + 512) = lo;
    }
    if (MODE == POLY) __syncthreads();
    // rows j, k along i: the mirror image of a symmetric result, or X's other orientation
    _Float16* out = HALF ? p.out0 + b * p.out0_b : p.out1 + b * p.out1_b;
    const int64_t kbs = HALF ? p.out0_kb : p.out1_kb;
    for (int f = wave; f < (BN / 16) * (BM / 32); f += WAVES) {
        const int rj = f / (BM / 32), ki = f % (BM / 32);
        if (HALF && i0 / 32 + ki <= j0 / 32 + rj / 2) continue;
        half8 hi, lo;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            _Float16 h, l;
            split(tile[(ki * 32 + k8 + q) * PITCH + rj * 16 + row] * (1.0f / SCALE), h, l);
            hi[q] = h; lo[q] = l;
        }
        _Float16* to = out + ((int64_t)(j0 / 16 + rj) * kbs + i0 / 32 + ki) * FRAG + lane * 8;
        *(half8*)to = hi; *(half8*)(to + 512) = lo;
    }
}

// i0, j0: the tile's first row and column
template <int BM, int BN, int WM, int WN, int NS, int MODE>
__device__ __forceinline__ void product_tile(const product& p, int i0, int j0, char* lds) {
    typedef staged<BM, BN, WM, WN, NS> L;
    constexpr int WAVES = L::WAVES, TM = WM / 16, TN = WN / 16, ROWS = L::ROWS, PITCH = L::PITCH, STAGE = L::STAGE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t b = blockIdx.z;
    const int64_t along = (int64_t)p.kb * FRAG;          // of a row of fragments
    const _Float16* P = p.P + b * p.P_b + i0 / 16 * along;
    const _Float16* Q = p.Q + b * p.Q_b + j0 / 16 * along;

    // a step's copies into a stage: one instruction of a wave moves 1 KB, a plane of a fragment
    auto copy = [&](int f, int k, int stage) {
        const int piece = f * WAVES + wave, r = piece >> 1, plane = piece & 1;
        const _Float16* from = (r < BM / 16 ? P + r * along : Q + (r - BM / 16) * along) + ((int64_t)k * FRAG + plane * (FRAG / 2));
        auto at = (const __attribute__((address_space(1))) char*)from;
        asm("" : "+s"(at));          // the same for the wave: stays in scalar registers
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(at + (uint32_t)(lane * 16)), (__attribute__((address_space(3))) void*)(lds + stage * STAGE + piece * 1024), 16, 0, 0);
    };
    constexpr int READS = 2 * (TM + TN), PRODUCTS = 3 * TM * TN;
    // The small products hi lo and lo hi have sums of their own: every addition to a long sum rounds it, and these are two of three.
    float4_ acc[TM][TN] = {}, small[TM][TN] = {};
    const int wi = wave / (BN / WN), wj = wave % (BN / WN);
    struct fragments { half8 h[TM + TN], l[TM + TN]; };          // of P, then of Q
    auto read = [&](fragments& f, int n, int stage) {
        const int r = n >> 1;
        const char* from = lds + stage * STAGE + (r < TM ? wi * TM + r : BM / 16 + wj * TN + r - TM) * 2048 + (n & 1) * 1024 + lane * 16;
        (n & 1 ? f.l : f.h)[r] = *(const half8*)from;
    };
    auto multiply = [&](const fragments& f, int n) {          // hi lo for all, lo hi for all, hi hi for all: no sum twice in a row
        const int kind = n / (TM * TN), i = n / TN % TM, j = n % TN;
        const bool p_lo = kind == 1, q_lo = kind == 0;
        float4_& sum = p_lo != q_lo ? small[i][j] : acc[i][j];
        sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(p_lo ? f.l[i] : f.h[i], q_lo ? f.l[TM + j] : f.h[TM + j], sum, 0, 0, 0);
    };
    int stage = 0;                // of the step to be read
    // this wave's copies for the step to be read have arrived, and with the barrier everyone's; its reads of the step before are done
    auto arrived = [&](auto later) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(later)::value * L::MOVES) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // While step k is multiplied from registers, step k + 1 is read from LDS and step k + NS is copied into the stage whose last readers
    // the barrier has seen finish; one read and half a copy to every few products, in this order.
    auto advance = [&](const fragments& now, fragments& next, int k, auto copies) {
        const int to = (stage + NS - 1) % NS, from = min(k + NS, p.kb - 1);          // (behind the end: the last step once more)
#pragma unroll
        for (int n = 0; n < READS; ++n) {
            read(next, n, stage);
            if (decltype(copies)::value && n % (READS / L::MOVES) == 0 && n / (READS / L::MOVES) < L::MOVES) copy(n / (READS / L::MOVES), from, to);
#pragma unroll
            for (int e = PRODUCTS * n / READS; e < PRODUCTS * (n + 1) / READS; ++e) multiply(now, e);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = (stage + 1) % NS;
    };
    fragments even, odd;
#pragma unroll
    for (int k = 0; k < NS - 1; ++k)
#pragma unroll
        for (int f = 0; f < L::MOVES; ++f) copy(f, min(k, p.kb - 1), k);
    arrived(number<NS - 2>());
#pragma unroll
    for (int n = 0; n < READS; ++n) read(even, n, 0);
#pragma unroll
    for (int f = 0; f < L::MOVES; ++f) copy(f, min(NS - 1, p.kb - 1), NS - 1);
    stage = 1;
    for (int k = 0; k + 2 < p.kb; k += 2) {          // (kb is even: sides are padded to 128)
        arrived(number<NS - 2>());
        advance(even, odd, k, flag<true>());
        arrived(number<NS - 2>());
        advance(odd, even, k + 1, flag<true>());
    }
    arrived(number<0>());
    advance(even, odd, p.kb - 2, flag<false>());
#pragma unroll
    for (int e = 0; e < PRODUCTS; ++e) multiply(odd, e);
    __syncthreads();
    // the tile through LDS, so that both orientations leave in whole fragments.  A lane holds rows 4 (lane / 16) + r of column lane % 16.
    float* tile = (float*)lds;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) tile[(wi * WM + i * 16 + (lane >> 4) * 4 + r) * PITCH + wj * WN + j * 16 + (lane & 15)] = acc[i][j][r] + small[i][j][r];
    __syncthreads();
    finish<BM, BN, WAVES, MODE>(p, tile, i0, j0);
}

// 256 x 128 in four waves of 128 x 64: a wave keeps the four column fragments of a step and lets the eight row fragments pass by, two
// ahead of their products; the next step's column fragments come in during the second half of a step, behind the one barrier.
// (With all fragments of two steps at hand the sums no longer fit the vector registers, and are carried to and fro.)
template <int MODE>
__device__ __forceinline__ void wide_tile(const product& p, int i0, int j0, char* lds) {
    typedef staged<256, 128, 128, 64, 3> L;
    constexpr int TM = 8, TN = 4, PITCH = L::PITCH, STAGE = L::STAGE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), wi = wave >> 1, wj = wave & 1;
    const int64_t b = blockIdx.z;
    const int64_t along = (int64_t)p.kb * FRAG;          // of a row of fragments
    const _Float16* P = p.P + b * p.P_b + i0 / 16 * along;
    const _Float16* Q = p.Q + b * p.Q_b + j0 / 16 * along;
    auto copy = [&](int f, int k, int stage) {
        const int piece = f * 4 + wave, r = piece >> 1, plane = piece & 1;
        const _Float16* from = (r < 16 ? P + r * along : Q + (r - 16) * along) + ((int64_t)k * FRAG + plane * (FRAG / 2));
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + lane * 8), (__attribute__((address_space(3))) void*)(lds + stage * STAGE + piece * 1024), 16, 0, 0);
    };
    struct fragment { half8 h, l; };
    auto read = [&](fragment& f, int r, int stage) {
        const char* from = lds + stage * STAGE + r * 2048 + lane * 16;
        f.h = *(const half8*)from;
        f.l = *(const half8*)(from + 1024);
    };
    float4_ acc[TM][TN] = {}, small[TM][TN] = {};          // small: as in product_tile
    fragment row[4], even[TN], odd[TN];
    int now = 0, next = 1, free = 2;          // stages
    auto step = [&](const fragment (&col)[TN], fragment (&coming)[TN], int k, auto more) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if (decltype(more)::value && i == TM / 2) {
                // this wave's copies for step k + 1 have arrived, and with the barrier everyone's; everyone is past step k - 1
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
            if (i + 2 < TM) read(row[(i + 2) & 3], wi * TM + i + 2, now);
            else if (decltype(more)::value) read(row[(i + 2) & 3], wi * TM + i + 2 - TM, next);
            if (decltype(more)::value && i >= TM / 2) {
                read(coming[i - TM / 2], 16 + wj * TN + i - TM / 2, next);
#pragma unroll
                for (int f = 0; f < 3; ++f) copy((i - TM / 2) * 3 + f, min(k + 2, p.kb - 1), free);          // (behind the end: the last step once more)
            }
            const fragment& r = row[i & 3];
#pragma unroll
            for (int j = 0; j < TN; ++j) small[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.h, col[j].l, small[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < TN; ++j) small[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.l, col[j].h, small[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.h, col[j].h, acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        const int was = now;
        now = next; next = free; free = was;
    };
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int f = 0; f < L::MOVES; ++f) copy(f, k, k);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L::MOVES) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(row[0], wi * TM, 0);
    read(row[1], wi * TM + 1, 0);
#pragma unroll
    for (int j = 0; j < TN; ++j) read(even[j], 16 + wj * TN + j, 0);
    auto pin = [&] {          // the sums stay in accumulation registers
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                asm volatile("" : "+a"(acc[i][j]));
                asm volatile("" : "+a"(small[i][j]));
            }
    };
    pin();
    for (int k = 0; k + 2 < p.kb; k += 2) {          // (kb is even: sides are padded to 128)
        step(even, odd, k, flag<true>());
        step(odd, even, k + 1, flag<true>());
        pin();
    }
    step(even, odd, p.kb - 2, flag<true>());
    step(odd, even, p.kb - 1, flag<false>());
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    float* tile = (float*)lds;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) tile[(wi * 128 + i * 16 + (lane >> 4) * 4 + r) * PITCH + wj * 64 + j * 16 + (lane & 15)] = acc[i][j][r] + small[i][j][r];
    __syncthreads();
    finish<256, 128, 4, MODE>(p, tile, i0, j0);
}

// Tiles of 128 x 128, two workgroups per CU; those that would be left for a last round that fills less than two thirds of the chip are
// cut into four.  Workgroups go round the eight dies by their index: each die gets a run of neighbouring tiles, so that its L2 cache
// serves their common operands.  2 x 1031 x 4099: A 55, Q 19, Q X 64 to 70 us, the latter 750 to 810 TFLOP/s of 16-bit products (1031 is padded to 1152,
// and its last round is short).
template <int MODE>
__global__ __launch_bounds__(256, 2) void k_orth_product(product p) {
    typedef staged<128, 128, 64, 64, 2> big;
    __shared__ __attribute__((aligned(16))) char lds[big::BYTES];
    constexpr bool HALF = MODE == GRAM || MODE == POLY;
    int t = blockIdx.x, quarter = -1, ti, tj;
    if (t < p.whole) {
        const int per = p.whole / 8;
        if (t < per * 8) t = t % 8 * per + t / 8;
    } else {
        quarter = (t - p.whole) & 3;
        t = p.whole + ((t - p.whole) >> 2);
    }
    if (HALF) below(t, ti, tj);
    else {          // in bands of eight rows of tiles
        const int band = t / (8 * p.tiles_j), r = t - band * 8 * p.tiles_j, rows = min(8, p.tiles_i - band * 8);
        ti = band * 8 + r % rows; tj = r / rows;
    }
    if (quarter < 0) product_tile<128, 128, 64, 64, 2, MODE>(p, ti * 128, tj * 128, lds);
    else {
        ti = ti * 2 + (quarter >> 1); tj = tj * 2 + (quarter & 1);
        if (HALF && tj > ti) return;
        product_tile<64, 64, 32, 32, 4, MODE>(p, ti * 64, tj * 64, lds);
    }
}

// Tiles of 256 x 128, one workgroup per CU, for results that fill the chip with them.  A wave's 128 x 64 need 24 reads of LDS for 96
// products; with 64 x 64 it is 16 for 48, and LDS is what they wait for.  `whole` tiles, the rest of them in 64 x 64, and 64 x 64 for
// the last 128 rows where the padded short side is an odd multiple of 128.  4096 x 8192: A 366, Q 192, Q X 626 us, 1130, 1070 and 1320 TFLOP/s of
// 16-bit products; the library's large product of 16-bit matrices reaches 1330 to 1420: bound by the matrix cores, 0.63 to 0.68 busy (and by what power they may draw).
template <int MODE>
__global__ __launch_bounds__(256, 1) void k_orth_wide(product p) {
    typedef staged<256, 128, 128, 64, 3> big;
    __shared__ __attribute__((aligned(16))) char lds[big::BYTES];
    constexpr bool HALF = MODE == GRAM || MODE == POLY;
    int t = blockIdx.x, ti, tj;
    const int cut = (p.tiles - p.whole) * 8;
    if (t >= p.whole + cut) {          // the last 128 rows
        t -= p.whole + cut;
        ti = p.tiles_i * 4 + (t & 1); tj = t >> 1;
        if (HALF && tj > ti) return;
        return product_tile<64, 64, 32, 32, 8, MODE>(p, ti * 64, tj * 64, lds);
    }
    int part = -1;
    if (t < p.whole) {
        const int per = p.whole / 8;
        if (t < per * 8) t = t % 8 * per + t / 8;
    } else {
        part = (t - p.whole) & 7;
        t = p.whole + ((t - p.whole) >> 3);
    }
    if (HALF) {          // row ti of tiles has 2 ti + 2 of them, ti (ti + 1) come before
        ti = (int)((sqrtf(4.0f * t + 1.0f) - 1.0f) * 0.5f);
        while ((ti + 1) * (ti + 2) <= t) ++ti;
        while (ti * (ti + 1) > t) --ti;
        tj = t - ti * (ti + 1);
    } else {          // in bands of four rows of tiles
        const int band = t / (4 * p.tiles_j), r = t - band * 4 * p.tiles_j, rows = min(4, p.tiles_i - band * 4);
        ti = band * 4 + r % rows; tj = r / rows;
    }
    if (part < 0) return wide_tile<MODE>(p, ti * 256, tj * 128, lds);
    ti = ti * 4 + (part >> 1); tj = tj * 2 + (part & 1);
    if (HALF && tj > ti) return;
    product_tile<64, 64, 32, 32, 8, MODE>(p, ti * 64, tj * 64, lds);
}

// ---- the same products where there are too few tiles, or too few steps along k, to fill the chip with staged ones ----------------------
// One 32 x 32 tile per workgroup, eight waves take every eighth step along k straight from memory: all their loads are on the way at
// once, nothing is staged and nothing waited for but the sum over the waves.  Every element comes from the L2 cache 32 times
// (m n k / 4 bytes in all), which is what bounds it from some 800^3 on.
// A = X X' of a short and long X has few tiles and many steps: they are split over workgroups, and the last of a tile's to finish sums
// what all have left, in their order, not in that of their coming (100 x 8000, all five steps: 208 -> 126 us).
// 512 x 512: 5 to 7 us a product, of which the launch and the sum over the waves are the most.
template <int MODE>
__global__ __launch_bounds__(512) void k_orth_direct(product p) {
    constexpr int WAVES = 8;
    __shared__ __attribute__((aligned(16))) float part[WAVES][4][256];
    __shared__ float tile[32][33];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t b = blockIdx.z;
    int ti, tj;
    const int tile_ = MODE == GRAM ? blockIdx.x / p.splits : blockIdx.x, share = MODE == GRAM ? blockIdx.x % p.splits : 0;
    if (MODE == GRAM || MODE == POLY) below(tile_, ti, tj);
    else {
        ti = tile_ % p.tiles_i; tj = tile_ / p.tiles_i;
    }
    const int first = MODE == GRAM ? (int)((int64_t)p.kb * share / p.splits) : 0, last = MODE == GRAM ? (int)((int64_t)p.kb * (share + 1) / p.splits) : p.kb;
    const _Float16* P = p.P + b * p.P_b + (int64_t)ti * 2 * p.kb * FRAG + lane * 8;
    const _Float16* Q = p.Q + b * p.Q_b + (int64_t)tj * 2 * p.kb * FRAG + lane * 8;
    float4_ acc[2][2] = {};
#pragma unroll 4
    for (int k = first + wave; k < last; k += WAVES) {
        half8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const _Float16* f = P + ((int64_t)i * p.kb + k) * FRAG;
            ph[i] = *(const half8*)f; pl[i] = *(const half8*)(f + 512);
            f = Q + ((int64_t)i * p.kb + k) * FRAG;
            qh[i] = *(const half8*)f; ql[i] = *(const half8*)(f + 512);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[i], ql[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[i], qh[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[i], qh[j], acc[i][j], 0, 0, 0);
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) *(float4_*)&part[wave][i * 2 + j][lane * 4] = acc[i][j];
    const int i0 = ti * 32, j0 = tj * 32;
    __syncthreads();
    float4_ v = {};
    if (wave < 4) {          // a wave sums a quarter
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += *(const float4_*)&part[w][wave][lane * 4];
    }
    if (MODE == GRAM && p.splits > 1) {
        // left where every die sees it (a die's L2 cache does not hold it back), 8 bytes at a time
        const int64_t at = b * (gridDim.x / p.splits) + tile_;
        uint64_t* mine = (uint64_t*)p.parts + ((at * p.splits + share) * 4 + wave) * 128 + lane * 2;
        if (wave < 4) {
            __hip_atomic_store(mine, (uint64_t)__float_as_uint(v[1]) << 32 | __float_as_uint(v[0]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(mine + 1, (uint64_t)__float_as_uint(v[3]) << 32 | __float_as_uint(v[2]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // every wave's own have arrived before the count says so: the barrier waits for none, the count for its wave's only
        }
        __shared__ uint32_t before;
        __syncthreads();
        if (threadIdx.x == 0) before = __hip_atomic_fetch_add(p.arrived + at, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if ((int)before + 1 < p.splits) return;
        if (threadIdx.x == 0) __hip_atomic_store(p.arrived + at, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (wave < 4) {
            v = float4_{};
            mine -= (int64_t)share * 512;
#pragma unroll 8
            for (int k = 0; k < p.splits; ++k) {
                const uint64_t lo = __hip_atomic_load(mine + k * 512, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), hi = __hip_atomic_load(mine + k * 512 + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                v += float4_{__uint_as_float((uint32_t)lo), __uint_as_float((uint32_t)(lo >> 32)), __uint_as_float((uint32_t)hi), __uint_as_float((uint32_t)(hi >> 32))};
            }
        }
    }
    if (wave < 4) {
        const int i = (wave >> 1) * 16 + (lane >> 4) * 4, j = (wave & 1) * 16 + (lane & 15);
        if (MODE == POLY) {
            // A[i + r][j] lies in the fragment of row j (A is symmetric): four neighbours
            const _Float16* A = p.A + b * p.out0_b + (((int64_t)(j0 / 16 + (wave & 1))) * p.out0_kb + ti) * FRAG + ((lane & 15) + 16 * (i >> 3)) * 8 + (i & 7);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[r] = fmaf(p.c, v[r] * (1.0f / SCALE), p.b * ((float)A[r] + (float)A[512 + r])) * SCALE;
                if (i0 + i + r == j0 + j) v[r] += p.a * (SCALE * SCALE);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) tile[i + r][j] = v[r];
    }
    __syncthreads();
    if (MODE == LAST) {
        emit<32, 32, 512>(p, b, &tile[0][0], 33, i0, j0);
        return;
    }
    if (wave >= 4 || (MODE != STEP && wave >= 2 && ti == tj)) return;
    // two fragments with rows i and two with rows j: the mirror image of a symmetric result, or X's other orientation
    const bool turned = wave >= 2;
    const int row = (wave & 1) * 16 + (lane & 15), k = (lane >> 4) * 8;
    half8 hi, lo;
#pragma unroll
    for (int r = 0; r < 8; ++r) { _Float16 h, l; split((turned ? tile[k + r][row] : tile[row][k + r]) * (1.0f / SCALE), h, l); hi[r] = h; lo[r] = l; }
    _Float16* out = turned && MODE == STEP ? p.out1 + b * p.out1_b : p.out0 + b * p.out0_b;
    const int64_t kbs = turned && MODE == STEP ? p.out1_kb : p.out0_kb;
    _Float16* to = out + (((int64_t)(turned ? j0 : i0) / 16 + (wave & 1)) * kbs + (turned ? ti : tj)) * FRAG + lane * 8;
    *(half8*)to = hi;
    *(half8*)(to + 512) = lo;
}

// ---- small matrices: all of it in one workgroup ----------------------------------------------------------------------------------------
// m <= 16 RB rows, n <= 128 JB columns.  Wave w owns 16 JB columns.  A result of the matrix cores leaves lane (q, c) = (lane / 16, lane % 16)
// with rows 16 I + 4 q + r of column c; as an operand over k = 32 s .. a lane needs eight k's, the same ones in both operands, in
// any order.  With the order {32 s + 4 q + r, 32 s + 16 + 4 q + r} the results of the blocks I = 2 s and 2 s + 1 are an operand as they
// stand: X goes from step to step in registers, and Q, being symmetric, is one as it comes out (with RB = 1 the products over rows
// are those of the matrix cores' 32-bit instruction, whose operands are the results as they stand: with so few terms to average over, 22 bits
// in them left 3 x 700 off by up to 3.7 times what 32-bit products are).  Only A = X X', which sums over columns, reads X in its other
// orientation, from the wave's own part of LDS.  X itself stays in 32 bits: here Q is without its a I, and X = a X + Q X.  Two barriers per step, one with RB = 1, where A's parts are summed.
// Bound by what one CU does in sequence, some 450 instructions per wave and step with RB = 2, JB = 4, and the way in and out (vector units 0.29 and 0.43
// busy below, waves wait half of their time).  8 x 512: 14.7 us (13.4 with 16-bit products throughout, which lost
// the precision said above), 512 x 29 with momentum and weight: 29.
struct small {
    source s;
    int32_t m, n, steps, turned, flat;          // flat: the rows of every array follow each other, they are read as one
    float a, b, c;
    void* out; const void* w; int out_type, w_type;
    int64_t out_b, out_r, w_b, w_r;
    float keep, gain;
};

// The way in and out: fours of the caller's rows, and through LDS into the lanes that work on them.  There a row of the short side has
// NP places, its columns swapped by row, so that neither order meets in one bank.
template <int NP> struct cells {
    float* at;
    int turned, cols;             // the caller's
    float per_col;
    __device__ __forceinline__ cells(float* at_, const small& p) : at(at_), turned(p.turned), cols(p.turned ? p.m : p.n), per_col(1.0f / (p.turned ? p.m : p.n)) {}
    __device__ __forceinline__ float& operator()(int i, int j) const { return at[i * NP + (j ^ (i & 31))]; }
    template <typename F> __device__ __forceinline__ void four(bool flat, int r, int c, F&& f) const {          // f(k, cell) for c .. c + 3
        if (flat) { r = (int)((c + 0.5f) * per_col); c -= r * cols; }          // (exact: fewer than 2^16 places)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f(k, turned ? (*this)(c, r) : (*this)(r, c));
            if (++c == cols && flat) { c = 0; ++r; }
        }
    }
};

template <int NP, int AT_ONCE>
__device__ __forceinline__ double way_in(const small& p, const cells<NP>& cell, int rows_used, bool first) {
    const int64_t b = blockIdx.x;
    const int rows = p.flat ? 1 : p.turned ? p.n : p.m, cols = p.flat ? p.m * p.n : p.turned ? p.m : p.n, per = (cols + 3) / 4;
    if (p.m < rows_used || p.n < NP) {
        for (int e = threadIdx.x; e < rows_used * NP / 4; e += 512) ((float4_*)cell.at)[e] = float4_{};
        __syncthreads();
    }
    double sum = 0.0;
    for (int e = threadIdx.x; e < rows * per; e += AT_ONCE * 512) {
        place at[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int f = e + k * 512, r = p.flat ? 0 : f / per;
            at[k].b = b; at[k].r = r; at[k].c = (f - r * per) * 4;
            at[k].n = f < rows * per ? min(4, cols - (int)at[k].c) : 0;
            at[k].load(p.s, first);
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (at[k].n <= 0) continue;
            at[k].move(p.s, first);
            cell.four(p.flat, (int)at[k].r, (int)at[k].c, [&](int t, float& to) {
                if (t < at[k].n) to = at[k].u[t];
                sum += (double)at[k].u[t] * at[k].u[t];
            });
        }
    }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    return sum;
}

template <int NP, int AT_ONCE>
__device__ __forceinline__ void way_out(const small& p, const cells<NP>& cell) {
    const int64_t b = blockIdx.x;
    const int rows = p.flat ? 1 : p.turned ? p.n : p.m, cols = p.flat ? p.m * p.n : p.turned ? p.m : p.n, per = (cols + 3) / 4;
    const float gain = p.gain / SCALE;
    for (int e = threadIdx.x; e < rows * per; e += AT_ONCE * 512) {
        float4_ w[AT_ONCE];
        int row[AT_ONCE], col[AT_ONCE], left[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int f = e + k * 512;
            row[k] = p.flat ? 0 : f / per; col[k] = (f - row[k] * per) * 4;
            left[k] = f < rows * per ? min(4, cols - col[k]) : 0;
            w[k] = float4_{};
            if (p.w) {
                const int64_t at = b * p.w_b + row[k] * p.w_r + col[k];
                if (left[k] >= 4) w[k] = load4(p.w, p.w_type, at);
                else for (int t = 0; t < left[k]; ++t) w[k][t] = load_elem(p.w, p.w_type, at + t);
            }
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (left[k] <= 0) continue;
            const int64_t at = b * p.out_b + row[k] * p.out_r + col[k];
            float4_ v = {};
            cell.four(p.flat, row[k], col[k], [&](int t, float& from) { if (t < left[k]) v[t] = from * gain; });
            if (p.w) for (int t = 0; t < 4; ++t) v[t] = fmaf(p.keep, w[k][t], v[t]);
            if (left[k] >= 4) store4(p.out, p.out_type, at, v);
            else for (int t = 0; t < left[k]; ++t) store_elem(p.out, p.out_type, at + t, v[t]);
        }
    }
}

// The arithmetic of a step on x, a lane's part of X (times SCALE) in the layout of the results.
template <int RB, int JB> struct rowwise {
    static constexpr int NWAVES = 8, NP = NWAVES * JB * 16, KB = JB / 2, S = RB == 1 ? 1 : RB / 2, TILES = RB * (RB + 1) / 2;
    typedef _Float16 columns[NWAVES][RB][KB][FRAG];          // X over columns, a part for each wave
    typedef float sums[NWAVES][TILES][256];                  // the tiles of A, as each wave has them
    typedef _Float16 matrix_[RB == 1 ? 1 : RB][S][RB == 1 ? 8 : FRAG];
    struct operand { half8 h[JB][S], l[JB][S]; };            // X over rows

    template <bool STORE> static __device__ __forceinline__ void operands(const float (&x)[JB][RB][4], operand& o, columns& xr, int wave, int q, int c) {
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
            for (int I = 0; I < RB; ++I)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    _Float16 h, l;
                    split(x[jb][I][r], h, l);
                    o.h[jb][I / 2][(I & 1) * 4 + r] = h;
                    o.l[jb][I / 2][(I & 1) * 4 + r] = l;
                    if constexpr (STORE) {
                        _Float16* to = &xr[wave][I][jb / 2][(4 * q + r + 16 * ((jb & 1) * 2 + (c >> 3))) * 8 + (c & 7)];
                        to[0] = h;
                        to[512] = l;
                    }
                }
    }
    // this wave's part of A, from its own part of xr
    static __device__ __forceinline__ void gram(float4_ (&acc)[TILES], const columns& xr, int wave, int lane) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) acc[t] = float4_{};
#pragma unroll
        for (int k = 0; k < KB; ++k) {
            half8 ph[RB], pl[RB];
#pragma unroll
            for (int I = 0; I < RB; ++I) { ph[I] = *(const half8*)&xr[wave][I][k][lane * 8]; pl[I] = *(const half8*)&xr[wave][I][k][512 + lane * 8]; }
#pragma unroll
            for (int I = 0; I < RB; ++I)
#pragma unroll
                for (int J = 0; J <= I; ++J) {
                    float4_& t = acc[I * (I + 1) / 2 + J];
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[I], pl[J], t, 0, 0, 0);
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[I], ph[J], t, 0, 0, 0);
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[I], ph[J], t, 0, 0, 0);
                }
        }
    }
    static __device__ __forceinline__ float4_ total(const sums& red, int t, int lane) {
        float4_ v = {};
#pragma unroll
        for (int w = 0; w < NWAVES; ++w) v += *(const float4_*)&red[w][t][lane * 4];
        return v;
    }
    // X = a X + (b A + c A A) X, A from everyone's sums: one barrier, and with RB > 1 a second one inside
    static __device__ __forceinline__ void update(const small& p, float (&x)[JB][RB][4], const operand& o, const float4_ (&acc)[TILES], sums& red, matrix_& am, int wave, int lane) {
        const int q = lane >> 4, c = lane & 15;
#pragma unroll
        for (int t = 0; t < TILES; ++t) *(float4_*)&red[wave][t][lane * 4] = acc[t];
        __syncthreads();
        if constexpr (RB == 1) {
            // A and Q are symmetric: what a lane holds of rows 4 q + r is an operand over those four k's as it stands, and so is x
            const float4_ a = total(red, 0, lane) * (1.0f / (SCALE * SCALE));
            float4_ t = {}, m;
#pragma unroll
            for (int r = 0; r < 4; ++r) t = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], a[r], t, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) m[r] = fmaf(p.c, t[r], p.b * a[r]);
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) {
                float4_ y = {};
#pragma unroll
                for (int r = 0; r < 4; ++r) y = __builtin_amdgcn_mfma_f32_16x16x4f32(m[r], x[jb][0][r], y, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[jb][0][r] = fmaf(p.a, x[jb][0][r], y[r]);
            }
        } else {
            for (int t = wave; t < TILES; t += NWAVES) {          // a wave sums a tile and writes it, and its mirror image, as operands
                const float4_ v = total(red, t, lane);
                int I = 0;
                while ((I + 1) * (I + 2) / 2 <= t) ++I;
                const int J = t - I * (I + 1) / 2;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    _Float16 h, l;
                    split(v[r] * (1.0f / SCALE), h, l);
                    const int i = 16 * I + 4 * q + r, j = 16 * J + c;
                    _Float16* to = &am[J][i >> 5][(c + 16 * ((i & 31) >> 3)) * 8 + (i & 7)];
                    to[0] = h; to[512] = l;
                    if (I != J) {
                        to = &am[I][j >> 5][(4 * q + r + 16 * ((j & 31) >> 3)) * 8 + (j & 7)];
                        to[0] = h; to[512] = l;
                    }
                }
            }
            __syncthreads();
            half8 ah[RB][S], al[RB][S], qh[RB][S], ql[RB][S];
#pragma unroll
            for (int I = 0; I < RB; ++I)
#pragma unroll
                for (int k = 0; k < S; ++k) { ah[I][k] = *(const half8*)&am[I][k][lane * 8]; al[I][k] = *(const half8*)&am[I][k][512 + lane * 8]; }
#pragma unroll
            for (int J = 0; J < RB; ++J)
#pragma unroll
                for (int I = 0; I < RB; ++I) {
                    float4_ t = {};
#pragma unroll
                    for (int k = 0; k < S; ++k) {
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[I][k], al[J][k], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[I][k], ah[J][k], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[I][k], ah[J][k], t, 0, 0, 0);
                    }
                    const int i = 16 * I + 4 * q;          // A[i + r][16 J + c] lies as row 16 J + c, columns i + r
                    const _Float16* from = &am[J][i >> 5][(c + 16 * ((i & 31) >> 3)) * 8 + (i & 7)];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        _Float16 h, l;
                        split(fmaf(p.c, t[r] * (1.0f / SCALE), p.b * ((float)from[r] + (float)from[512 + r])), h, l);
                        qh[J][I / 2][(I & 1) * 4 + r] = h;
                        ql[J][I / 2][(I & 1) * 4 + r] = l;
                    }
                }
#pragma unroll
            for (int jb = 0; jb < JB; ++jb)
#pragma unroll
                for (int I = 0; I < RB; ++I) {
                    float4_ t = {};
#pragma unroll
                    for (int k = 0; k < S; ++k) {
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[I][k], o.l[jb][k], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql[I][k], o.h[jb][k], t, 0, 0, 0);
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[I][k], o.h[jb][k], t, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[jb][I][r] = fmaf(p.a, x[jb][I][r], t[r] * (1.0f / SCALE));
                }
        }
    }
    // between the caller's order and the lanes'
    static __device__ __forceinline__ void pick(float (&x)[JB][RB][4], const cells<NP>& cell, double inv, int wave, int q, int c) {
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
            for (int I = 0; I < RB; ++I)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[jb][I][r] = (float)(cell(16 * I + 4 * q + r, (wave * JB + jb) * 16 + c) * inv);
    }
    static __device__ __forceinline__ void put(const float (&x)[JB][RB][4], const cells<NP>& cell, int wave, int q, int c) {
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
            for (int I = 0; I < RB; ++I)
#pragma unroll
                for (int r = 0; r < 4; ++r) cell(16 * I + 4 * q + r, (wave * JB + jb) * 16 + c) = x[jb][I][r];
    }
};

template <int RB, int JB>
__global__ __launch_bounds__(512) void k_orth_small(small p) {
    typedef rowwise<RB, JB> R;
    __shared__ __attribute__((aligned(16))) typename R::columns xr;
    __shared__ __attribute__((aligned(16))) typename R::sums red[RB == 1 ? 2 : 1];          // (RB = 1, one barrier: every other step the other one)
    __shared__ __attribute__((aligned(16))) typename R::matrix_ am;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), q = lane >> 4, c = lane & 15;
    const cells<R::NP> cell((float*)&xr[0][0][0][0], p);
    double sum = way_in<R::NP, 8>(p, cell, RB * 16, true);
    double* sums = (double*)red;
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < R::NWAVES; ++w) sum += sums[w];
    float x[JB][RB][4];
    R::pick(x, cell, sum != 0.0 ? (double)SCALE / sqrt(sum) : 0.0, wave, q, c);          // (NaN != 0)
    __syncthreads();
    for (int step = 0; step < p.steps; ++step) {
        typename R::operand o;
        float4_ acc[R::TILES];
        R::template operands<true>(x, o, xr, wave, q, c);
        R::gram(acc, xr, wave, lane);
        R::update(p, x, o, acc, red[RB == 1 ? step & 1 : 0], am, wave, lane);
    }
    __syncthreads();          // (the last reads of xr)
    R::put(x, cell, wave, q, c);
    __syncthreads();
    way_out<R::NP, 8>(p, cell);
}

// ---- short sides of up to 64 with a long one: a workgroup per 128 JB columns ("slab"), a launch per step ---------------------------------------
// Slab s leaves its part of A behind each launch; the next one sums all slabs' parts for itself, makes Q, moves its part of X on.
// X waits in memory between the launches, in 32 bits and in the order of the lanes.  Seven launches instead of seventeen, each bound by
// its way to the caches and back.  All five steps of 8 x 8000: 35 to 38 us (157 with a launch per product), 30 x 8000: 51, 8 x 100000: 73.
struct slabs {
    const double* partials; int32_t n_partials;
    float* x;                     // [batch][slab][JB * RB][512 lanes][4]
    float* parts[2];              // [batch][slab][TILES][256]: read and written in turn
    int32_t step;                 // 0: X from the gradient;  p.steps: the result
};

template <int RB, int JB>
__global__ __launch_bounds__(512) void k_orth_slab(small p, slabs sl) {
    typedef rowwise<RB, JB> R;
    __shared__ __attribute__((aligned(16))) typename R::columns xr;
    __shared__ __attribute__((aligned(16))) typename R::sums red;
    __shared__ __attribute__((aligned(16))) typename R::matrix_ am;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), q = lane >> 4, c = lane & 15;
    const int slab = blockIdx.y, n_slabs = gridDim.y, j0 = slab * R::NP;
    const int64_t b = blockIdx.x, part = (b * n_slabs + slab) * R::TILES * 256;
    // from here on the slab is a matrix of its own
    p.n = min(p.n - j0, R::NP);
    const auto at = [&](int64_t row) { return p.turned ? j0 * row : j0; };
    const int size = p.s.dtype == 0 ? 4 : 2, w_size = p.w_type == 0 ? 4 : 2, out_size = p.out_type == 0 ? 4 : 2;
    p.s.g = (const char*)p.s.g + at(p.s.g_r) * size;
    if (p.s.m) p.s.m_out += at(p.s.o_r);
    if (p.w) p.w = (const char*)p.w + at(p.w_r) * w_size;
    p.out = (char*)p.out + at(p.out_r) * out_size;
    const cells<R::NP> cell((float*)&xr[0][0][0][0], p);
    float x[JB][RB][4];
    float4_* mine = (float4_*)sl.x + (b * n_slabs + slab) * (JB * RB) * 512 + threadIdx.x;
    typename R::operand o;
    float4_ acc[R::TILES];
    if (sl.step == 0) {
        way_in<R::NP, 8>(p, cell, RB * 16, false);
        double sum = 0.0;
        for (int k = lane; k < sl.n_partials; k += 64) sum += sl.partials[b * sl.n_partials + k];
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
        __syncthreads();
        R::pick(x, cell, sum != 0.0 ? (double)SCALE / sqrt(sum) : 0.0, wave, q, c);
        __syncthreads();
    } else {
#pragma unroll
        for (int e = 0; e < JB * RB; ++e) {
            const float4_ v = mine[e * 512];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[e / RB][e % RB][r] = v[r];
        }
        const float* from = sl.parts[(sl.step + 1) & 1] + b * n_slabs * R::TILES * 256 + lane * 4;
#pragma unroll
        for (int t = 0; t < R::TILES; ++t) acc[t] = float4_{};
        for (int k = wave; k < n_slabs; k += R::NWAVES) {
#pragma unroll
            for (int t = 0; t < R::TILES; ++t) acc[t] += *(const float4_*)(from + ((int64_t)k * R::TILES + t) * 256);
        }
        R::template operands<false>(x, o, xr, wave, q, c);
        R::update(p, x, o, acc, red, am, wave, lane);
        if (sl.step == p.steps) {
            R::put(x, cell, wave, q, c);
            __syncthreads();
            return way_out<R::NP, 8>(p, cell);
        }
    }
#pragma unroll
    for (int e = 0; e < JB * RB; ++e) mine[e * 512] = float4_{x[e / RB][e % RB][0], x[e / RB][e % RB][1], x[e / RB][e % RB][2], x[e / RB][e % RB][3]};
    R::template operands<true>(x, o, xr, wave, q, c);
    R::gram(acc, xr, wave, lane);
    __syncthreads();          // (the last reads of red)
#pragma unroll
    for (int t = 0; t < R::TILES; ++t) *(float4_*)&red[wave][t][lane * 4] = acc[t];
    __syncthreads();
    for (int t = wave; t < R::TILES; t += R::NWAVES) *(float4_*)(sl.parts[sl.step & 1] + part + t * 256 + lane * 4) = R::total(red, t, lane);
}

}  // namespace dlo
