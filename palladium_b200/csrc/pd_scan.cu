// pd_scan.cu -- the CUDA kernels of the state-space families: a short causal
// convolution over a sequence's tokens and the selective scan, the exact
// integration of an ensemble of driven linear systems
//     h' = A h + B(t) x(t),   y = C(t) h + D x
// over steps of input-dependent length, one trajectory per (sequence, channel).
// Compiled once per math mode like pd_kernels.cu: SAFE and RELAXED use the
// library's expf / log1pf and IEEE division, FAST the approximate ones.
//
// Everything is computed in float32 whatever the element type; a result is
// rounded once, where it is stored.
#include "pd_scan.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/palladium_cuda.h"

#ifndef PD_MODE
#error "PD_MODE must be 0 (SAFE), 1 (RELAXED) or 2 (FAST)"
#endif
#if PD_MODE == 0
#define PD_SCAN_TABLE pd_scan_table_safe
#elif PD_MODE == 1
#define PD_SCAN_TABLE pd_scan_table_relaxed
#else
#define PD_SCAN_TABLE pd_scan_table_fast
#endif

namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kStates = 4;     // states per thread

// ---------------------------------------------------------------------------
// elements
// ---------------------------------------------------------------------------
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// V consecutive elements, as stored; V > 1 means one aligned access of 8 or 16 bytes
template <class T, int V> struct Vec { T e[V]; };
template <int V, class T>
__device__ __forceinline__ Vec<T, V> fetch(const T* p) {
    Vec<T, V> r;
    if constexpr (V == 1) r.e[0] = p[0];
    else if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(r.e) = *reinterpret_cast<const uint4*>(p);
    else *reinterpret_cast<uint2*>(r.e) = *reinterpret_cast<const uint2*>(p);
    return r;
}
template <int V, class T>
__device__ __forceinline__ void widen(const Vec<T, V>& r, float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = load1(&r.e[i]);
}
template <int V, class T>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) { widen(fetch<V>(p), v); }
template <int V, class T>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) store1(&r.e[i], v[i]);
    if constexpr (V == 1) p[0] = r.e[0];
    else if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.e);
    else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(r.e);
}

// ---------------------------------------------------------------------------
// functions
// ---------------------------------------------------------------------------
__device__ __forceinline__ float exp_(float v) {
#if PD_MODE == 2
    return __expf(v);
#else
    return expf(v);
#endif
}
__device__ __forceinline__ float sigmoid_(float v) {
#if PD_MODE == 2
    return __fdividef(1.0f, 1.0f + __expf(-v));
#else
    return 1.0f / (1.0f + expf(-v));
#endif
}
// log(1 + e^v) = max(v, 0) + log1p(e), e = e^-|v| <= 1, without cancellation: a step size of 1e-3 is as exact
// as one of 10.  FAST sums log1p(e) = 2 artanh(s), s = e / (2 + e) <= 1/3, as 2 s (1 + s^2/3 + .. + s^12/13):
// the next term is below 2e-8 of the sum, and no branch is taken.
__device__ __forceinline__ float log1p_unit(float e) {
#if PD_MODE == 2
    const float s = __fdividef(e, 2.0f + e), q = s * s;
    float p = 1.0f / 13.0f;
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    return fmaf(2.0f * s, q * p, 2.0f * s);
#else
    return log1pf(e);
#endif
}
__device__ __forceinline__ float softplus_(float v) { return fmaxf(v, 0.0f) + log1p_unit(exp_(-fabsf(v))); }
// the same with its slope, 1 / (1 + e^-v)
__device__ __forceinline__ float softplus_(float v, float& slope) {
    const float e = exp_(-fabsf(v));
#if PD_MODE == 2
    const float r = __fdividef(1.0f, 1.0f + e);
#else
    const float r = 1.0f / (1.0f + e);
#endif
    slope = v >= 0.0f ? r : e * r;
    return fmaxf(v, 0.0f) + log1p_unit(e);
}

// ---------------------------------------------------------------------------
// pairs: one instruction, and one issue slot, for two float32 operations
// ---------------------------------------------------------------------------
typedef unsigned long long pair_t;     // two float32 in one 64-bit register
__device__ __forceinline__ pair_t pack(float x, float y) {
    pair_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void unpack(pair_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
    pair_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
    pair_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
// a b + c: one rounding, except under SAFE, which keeps the product's own
__device__ __forceinline__ pair_t mad2(pair_t a, pair_t b, pair_t c) {
#if PD_MODE == 0
    return add2(mul2(a, b), c);
#else
    pair_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
#endif
}

__device__ __forceinline__ float halves(pair_t v) {
    float x, y;
    unpack(v, x, y);
    return x + y;
}
// V elements as pairs (one element: its pair's other half is zero)
template <int V> constexpr int kPairs = (V + 1) / 2;
template <int V>
__device__ __forceinline__ void pair_up(const float (&v)[V], pair_t (&p)[kPairs<V>]) {
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) p[i] = pack(v[2 * i], 2 * i + 1 < V ? v[2 * i + 1 < V ? 2 * i + 1 : 0] : 0.0f);
}
template <int V>
__device__ __forceinline__ void part(const pair_t (&p)[kPairs<V>], float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
        float x, y;
        unpack(p[i], x, y);
        v[2 * i] = x;
        if (2 * i + 1 < V) v[2 * i + 1 < V ? 2 * i + 1 : 0] = y;
    }
}

// ---------------------------------------------------------------------------
// sequences
// ---------------------------------------------------------------------------
__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t rows) { return v < 0 ? 0 : (v > rows ? rows : v); }
__device__ __forceinline__ void bounds_of(const PdTokens& t, int64_t s, int64_t& begin, int64_t& end) {
    if (!t.offsets) {
        begin = s * t.length;
        end = begin + t.length;
        return;
    }
    begin = clamp_row(t.offsets[s], t.rows);
    end = clamp_row(t.offsets[s + 1], t.rows);
    if (end < begin) end = begin;
}
// The sequence that has `row`: true with its bounds, or false (rows before the first or behind the last one).
__device__ __forceinline__ bool sequence_of(const PdTokens& t, int64_t row, int64_t& s, int64_t& begin, int64_t& end) {
    if (!t.offsets) {
        s = row / t.length;
        begin = s * t.length;
        end = begin + t.length;
        return true;
    }
    int64_t lo = 0, hi = t.seqs;   // the last s with offsets[s] <= row
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if ((int64_t)t.offsets[mid] <= row) lo = mid + 1; else hi = mid;
    }
    s = lo - 1;
    if (s < 0) return false;
    bounds_of(t, s, begin, end);
    return begin <= row && row < end;
}
// Rows of no sequence in a packed call: those before the first one, [0, head), and behind the last one, [tail, rows).
__device__ __forceinline__ void free_rows(const PdTokens& t, int64_t& head, int64_t& tail) {
    head = clamp_row(t.offsets[0], t.rows);
    tail = clamp_row(t.offsets[t.seqs], t.rows);
    if (tail < head) tail = head;
}
// a block's share, one of `parts`, of n elements set to zero
template <class T>
__device__ __forceinline__ void clear_share(T* p, int64_t n, int64_t part, int64_t parts) {
    constexpr int V = 16 / sizeof(T);
    const int64_t share = ((n + parts - 1) / parts + V - 1) / V * V, from = part * share;
    if (from >= n) return;
    const int64_t to = from + share < n ? from + share : n;
    const int64_t up = from + (int64_t)(-reinterpret_cast<uintptr_t>(p + from) & 15) / (int64_t)sizeof(T);
    const int64_t low = up < to ? up : to, high = low + (to - low) / V * V;      // 16-byte stores in [low, high)
    for (int64_t i = from + threadIdx.x; i < low; i += blockDim.x) store1(p + i, 0.0f);
    for (int64_t i = low + (int64_t)threadIdx.x * V; i < high; i += (int64_t)blockDim.x * V)
        *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
    for (int64_t i = high + threadIdx.x; i < to; i += blockDim.x) store1(p + i, 0.0f);
}
template <class T>
__device__ __forceinline__ void clear_free_rows(const PdTokens& t, int64_t channels, T* p, int64_t part, int64_t parts) {
    int64_t head, tail;
    free_rows(t, head, tail);
    clear_share(p, head * channels, part, parts);
    clear_share(p + tail * channels, (t.rows - tail) * channels, part, parts);
}
// where the state entering each chunk of a sequence is kept
__device__ __forceinline__ int64_t first_chunk(const PdTokens& t, int64_t s, int64_t begin) {
    return t.offsets ? begin / PD_SCAN_CHUNK + s : s * ((t.length + PD_SCAN_CHUNK - 1) / PD_SCAN_CHUNK);
}

// ===========================================================================
// causal convolution:  y_t = act(bias + sum_j w[W-1-j] x_{t-j})
// One thread owns V channels and a run of consecutive rows; the last W - 1
// inputs stay in registers, so a row is read once apart from the run's halo.
// Bound: the latency of its rows.  8 x 2048 x 4096 in bf16 take 58 us, where memory,
// 2 bytes in and 2 out per element, asks for 41 and two special-function
// operations for 30; a warp waits on loads 8 of every 13 cycles.  So what matters
// is to keep rows in flight: four of them per thread, with four blocks of 256
// threads on an SM (82 us with two blocks and the next four rows fetched ahead, 76
// with eight channels per thread).  At their 64 registers width 4 spills 44 bytes in
// bf16 and 72 in float32.
// ===========================================================================
// the taps and the bias of V channels, as 16-byte vectors where the channels are
template <int W, int V>
__device__ __forceinline__ void conv_parameters(const PdConvArgs& a, int64_t c, pair_t (&w)[W][kPairs<V>], pair_t (&b)[kPairs<V>]) {
    float flat[V * W], bias[V];
    if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V * W / 4; ++i) {
            const float4 q = reinterpret_cast<const float4*>(a.weight + c * W)[i];
            flat[4 * i] = q.x; flat[4 * i + 1] = q.y; flat[4 * i + 2] = q.z; flat[4 * i + 3] = q.w;
        }
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float4 q = a.bias ? reinterpret_cast<const float4*>(a.bias + c)[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            bias[4 * i] = q.x; bias[4 * i + 1] = q.y; bias[4 * i + 2] = q.z; bias[4 * i + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V * W; ++i) flat[i] = a.weight[c * W + i];
#pragma unroll
        for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[c + v] : 0.0f;
    }
    pair_up<V>(bias, b);
#pragma unroll
    for (int k = 0; k < W; ++k) {
        float tap[V];
#pragma unroll
        for (int v = 0; v < V; ++v) tap[v] = flat[v * W + k];
        pair_up<V>(tap, w[k]);
    }
}

template <int V, class T>
__device__ __forceinline__ void widen(const Vec<T, V>& r, pair_t (&p)[kPairs<V>]) {
    float v[V];
    widen(r, v);
    pair_up<V>(v, p);
}
template <int V, class T>
__device__ __forceinline__ void load(const T* at, pair_t (&p)[kPairs<V>]) { widen(fetch<V>(at), p); }
template <int V, class T>
__device__ __forceinline__ void store(T* at, const pair_t (&p)[kPairs<V>]) {
    float v[V];
    part<V>(p, v);
    store<V>(at, v);
}

// the W - 1 inputs before `row`, oldest first
template <class T, int W, int V>
__device__ __forceinline__ void conv_window(const PdConvArgs& a, const T* x, int64_t s, int64_t begin, int64_t row,
                                            int64_t c, pair_t (&win)[W - 1][kPairs<V>]) {
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t r = row - (W - 1) + i;
        if (r >= begin) {
            load<V>(x + r * a.channels + c, win[i]);
        } else if (a.initial) {
            load<V>((const T*)a.initial + (s * (W - 1) + (W - 1) + (r - begin)) * a.channels + c, win[i]);
        } else {
#pragma unroll
            for (int p = 0; p < kPairs<V>; ++p) win[i][p] = 0;
        }
    }
}
template <int W, int P>
__device__ __forceinline__ void slide(pair_t (&win)[W][P], const pair_t (&now)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i + 1 < W; ++i) win[i][p] = win[i + 1][p];
        win[W - 1][p] = now[p];
    }
}
// bias + sum_j w[j] (window, now)[j]
template <int W, int P>
__device__ __forceinline__ void convolve(const pair_t (&w)[W][P], const pair_t (&b)[P], const pair_t (&win)[W - 1][P],
                                         const pair_t (&now)[P], pair_t (&pre)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        pre[p] = b[p];
#pragma unroll
        for (int i = 0; i < W - 1; ++i) pre[p] = mad2(w[i][p], win[i][p], pre[p]);
        pre[p] = mad2(w[W - 1][p], now[p], pre[p]);
    }
}
template <int V>
__device__ __forceinline__ void silu(const pair_t (&pre)[kPairs<V>], float (&out)[V]) {
    part<V>(pre, out);
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] *= sigmoid_(out[v]);
}

template <class T, int W, int V, bool SILU>
__global__ void __launch_bounds__(256, 4) pd_causal_conv_kernel(PdConvArgs a) {
    constexpr int P = kPairs<V>;
    const int64_t lanes = (a.channels + V - 1) / V;
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t job = id / lanes, c = id % lanes * V;
    const int64_t runs = (a.tok.rows + a.run - 1) / a.run;
    const T* x = (const T*)a.x;
    const float none[V] = {};
    if (job >= runs) {
        // one more job per sequence: an empty one hands its carried-in inputs on
        const int64_t s = job - runs;
        if (!a.final_state || s >= a.tok.seqs) return;
        int64_t begin, end;
        bounds_of(a.tok, s, begin, end);
        if (begin < end) return;
        for (int i = 0; i < W - 1; ++i) {
            const int64_t at = (s * (W - 1) + i) * a.channels + c;
            float v[V] = {};
            if (a.initial) load<V>((const T*)a.initial + at, v);
            store<V>((T*)a.final_state + at, v);
        }
        return;
    }
    pair_t w[W][P], b[P], win[W - 1][P];
    conv_parameters<W, V>(a, c, w, b);
    int64_t row = job * a.run;
    const int64_t stop = row + a.run < a.tok.rows ? row + a.run : a.tok.rows;
    while (row < stop) {
        int64_t s, begin, end;
        if (!sequence_of(a.tok, row, s, begin, end)) {
            store<V>((T*)a.y + row * a.channels + c, none);
            ++row;
            continue;
        }
        conv_window<T, W, V>(a, x, s, begin, row, c, win);
        const int64_t upto = end < stop ? end : stop;
        const T* from = x + row * a.channels + c;
        T* to = (T*)a.y + row * a.channels + c;
        auto step = [&](const Vec<T, V>& got) {
            pair_t now[P], pre[P];
            widen(got, now);
            convolve<W, P>(w, b, win, now, pre);
            slide<W - 1, P>(win, now);
            if (SILU) {
                float out[V];
                silu<V>(pre, out);
                store<V>(to, out);
            } else {
                store<V>(to, pre);
            }
            to += a.channels;
        };
        constexpr int F = 4;
        const int blocks = (int)((upto - row) / F);
        for (int k = 0; k < blocks; ++k) {
            Vec<T, V> got[F];
#pragma unroll
            for (int i = 0; i < F; ++i) got[i] = fetch<V>(from + i * a.channels);
            from += F * a.channels;
#pragma unroll
            for (int i = 0; i < F; ++i) step(got[i]);
        }
        for (row += (int64_t)blocks * F; row < upto; ++row, from += a.channels) step(fetch<V>(from));
        if (row == end && a.final_state)
#pragma unroll
            for (int i = 0; i < W - 1; ++i)
                store<V>((T*)a.final_state + (s * (W - 1) + i) * a.channels + c, win[i]);
    }
}

// one token per sequence: the window comes from and goes to the state (which may be the same memory)
template <class T, int W, int V>
__global__ void __launch_bounds__(128) pd_causal_conv_step_kernel(PdConvArgs a) {
    constexpr int P = kPairs<V>;
    const int lanes = (int)((a.channels + V - 1) / V), lane = blockIdx.x * blockDim.x + threadIdx.x;
    if (lane >= lanes) return;
    const int64_t c = (int64_t)lane * V;
    for (int64_t s = blockIdx.y; s < a.tok.seqs; s += gridDim.y) {
        pair_t win[W - 1][P], now[P], pre[P], w[W][P], b[P];
        const int64_t at = s * (W - 1) * a.channels + c;
#pragma unroll
        for (int i = 0; i < W - 1; ++i) load<V>((const T*)a.initial + at + i * a.channels, win[i]);
        load<V>((const T*)a.x + s * a.channels + c, now);
        conv_parameters<W, V>(a, c, w, b);
        convolve<W, P>(w, b, win, now, pre);
        if (a.silu) {
            float out[V];
            silu<V>(pre, out);
            store<V>((T*)a.y + s * a.channels + c, out);
        } else {
            store<V>((T*)a.y + s * a.channels + c, pre);
        }
        slide<W - 1, P>(win, now);
#pragma unroll
        for (int i = 0; i < W - 1; ++i) store<V>((T*)a.final_state + at + i * a.channels, win[i]);
    }
}

// Gradients.  With g_t = dy_t act'(pre_t):
//   dx_t = sum_j w[W-1-j] g_{t+j},   dw[W-1-j] = sum_t x_{t-j} g_t,   dbias = sum_t g_t
// A thread walks its run and W - 1 rows beyond it, and keeps the W gradients of dx still open; sums of
// dw and dbias stay in registers, then go to one partial per block, which a second launch adds up in order.
template <class T, int W, int V, bool SILU>
__global__ void __launch_bounds__(256, 2) pd_causal_conv_grad_kernel(PdConvArgs a) {
    constexpr int P = kPairs<V>;
    const int64_t lanes = (a.channels + V - 1) / V;
    // blockDim.x threads across channels, blockDim.y across runs; blockIdx.x channel blocks, blockIdx.y row blocks
    const int64_t lane = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t c = lane * V;
    const bool active = lane < lanes;
    const T* x = (const T*)a.x;
    const T* dy = (const T*)a.dy;
    const float none[V] = {};
    pair_t w[W][P], b[P], dw[W][P], db[P];
    if (active) conv_parameters<W, V>(a, c, w, b);
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][p] = 0;
        db[p] = 0;
    }
    const int64_t runs = (a.tok.rows + a.run - 1) / a.run;
    const int64_t jobs = runs + (a.dinitial ? a.tok.seqs : 0);
    for (int64_t job = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; active && job < jobs;
         job += (int64_t)gridDim.y * blockDim.y) {
        if (job >= runs) {
            // an empty sequence hands the gradient of its carried-out inputs back
            const int64_t s = job - runs;
            int64_t begin, end;
            bounds_of(a.tok, s, begin, end);
            if (begin < end) continue;
            for (int i = 0; i < W - 1; ++i) {
                const int64_t at = (s * (W - 1) + i) * a.channels + c;
                float v[V] = {};
                if (a.dfinal) load<V>((const T*)a.dfinal + at, v);
                store<V>((T*)a.dinitial + at, v);
            }
            continue;
        }
        int64_t row = job * a.run;
        const int64_t stop = row + a.run < a.tok.rows ? row + a.run : a.tok.rows;
        while (row < stop) {
            int64_t s, begin, end;
            if (!sequence_of(a.tok, row, s, begin, end)) {
                store<V>((T*)a.dx + row * a.channels + c, none);
                ++row;
                continue;
            }
            pair_t win[W - 1][P], open[W][P];   // open[j]: gradient of the input j rows back from the current one
            conv_window<T, W, V>(a, x, s, begin, row, c, win);
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int p = 0; p < P; ++p) open[j][p] = 0;
            const int64_t mine = end < stop ? end : stop;                        // rows whose sums belong here
            const int64_t upto = mine + (W - 1) < end ? mine + (W - 1) : end;    // rows whose g they need
            const int64_t first = row;
            const T* from_x = x + row * a.channels + c;
            const T* from_g = dy + row * a.channels + c;
            T* to = (T*)a.dx + (row - (W - 1)) * a.channels + c;                 // where the input W - 1 rows back goes
            auto step = [&](const Vec<T, V>& got_x, const Vec<T, V>& got_g, bool counts) {
                pair_t now[P], g[P];
                widen(got_x, now);
                if (SILU) {
                    pair_t pre[P];
                    float v[V], q[V];
                    convolve<W, P>(w, b, win, now, pre);
                    part<V>(pre, q);
                    widen(got_g, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float sig = sigmoid_(q[i]);
                        v[i] *= sig * (1.0f + q[i] * (1.0f - sig));
                    }
                    pair_up<V>(v, g);
                } else {
                    widen(got_g, g);
                }
#pragma unroll
                for (int p = 0; p < P; ++p) {
#pragma unroll
                    for (int j = W - 1; j > 0; --j) open[j][p] = mad2(w[W - 1 - j][p], g[p], open[j - 1][p]);
                    open[0][p] = mul2(w[W - 1][p], g[p]);
                    if (counts) {
                        db[p] = add2(db[p], g[p]);
#pragma unroll
                        for (int i = 0; i < W - 1; ++i) dw[i][p] = mad2(win[i][p], g[p], dw[i][p]);
                        dw[W - 1][p] = mad2(now[p], g[p], dw[W - 1][p]);
                    }
                }
                slide<W - 1, P>(win, now);
            };
            // the first W - 1 rows: the inputs before them are carried in, or another run's
            auto edge = [&](bool counts) {
                step(fetch<V>(from_x), fetch<V>(from_g), counts);
                const int64_t done = row - (W - 1);
                if (done >= first) store<V>(to, open[W - 1]);
                else if (done < begin && first == begin && a.dinitial) {
                    // (a carried-in input that is carried out again is still open at the end, below)
                    store<V>((T*)a.dinitial + (s * (W - 1) + (done - begin) + (W - 1)) * a.channels + c, open[W - 1]);
                }
                ++row;
                from_x += a.channels;
                from_g += a.channels;
                to += a.channels;
            };
            const int64_t head = first + (W - 1) < mine ? first + (W - 1) : mine;
            while (row < head) edge(true);
            constexpr int F = 4;
            const int blocks = (int)((mine - row) / F);
            for (int k = 0; k < blocks; ++k) {
                Vec<T, V> got_x[F], got_g[F];
#pragma unroll
                for (int i = 0; i < F; ++i) {
                    got_x[i] = fetch<V>(from_x + i * a.channels);
                    got_g[i] = fetch<V>(from_g + i * a.channels);
                }
                from_x += F * a.channels;
                from_g += F * a.channels;
#pragma unroll
                for (int i = 0; i < F; ++i) {
                    step(got_x[i], got_g[i], true);
                    store<V>(to, open[W - 1]);
                    to += a.channels;
                }
            }
            row += (int64_t)blocks * F;
            while (row < upto) edge(row < mine);
            if (row == end) {
                // the sequence ends here: the inputs still open are complete, and were carried out
#pragma unroll
                for (int j = W - 2; j >= 0; --j) {
                    const int64_t r = end - 1 - j;
                    float v[V];
                    part<V>(open[j], v);
                    if (a.dfinal) {
                        float f[V];
                        load<V>((const T*)a.dfinal + (s * (W - 1) + (W - 2 - j)) * a.channels + c, f);
#pragma unroll
                        for (int u = 0; u < V; ++u) v[u] += f[u];
                    }
                    if (r >= first && r < mine) store<V>((T*)a.dx + r * a.channels + c, v);
                    else if (r < begin && first == begin && a.dinitial)
                        store<V>((T*)a.dinitial + (s * (W - 1) + (r - begin) + (W - 1)) * a.channels + c, v);
                }
            }
            row = mine;
        }
    }
    // block sums, in the order of the runs
    extern __shared__ float sums[];   // (blockDim.y, blockDim.x, V)
#pragma unroll
    for (int k = 0; k <= W; ++k) {
        float mine[V];
        part<V>(k < W ? dw[k < W ? k : 0] : db, mine);
#pragma unroll
        for (int v = 0; v < V; ++v) sums[(threadIdx.y * blockDim.x + threadIdx.x) * V + v] = mine[v];
        __syncthreads();
        if (threadIdx.y == 0 && active)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float total = 0.0f;
                for (int y = 0; y < (int)blockDim.y; ++y) total += sums[(y * blockDim.x + threadIdx.x) * V + v];
                a.partial[((int64_t)blockIdx.y * a.channels + c + v) * (W + 1) + k] = total;
            }
        __syncthreads();
    }
}

template <int W>
__global__ void __launch_bounds__(128) pd_causal_conv_sum_kernel(PdConvArgs a) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.channels * (W + 1)) return;
    float total = 0.0f;
    for (int64_t b = 0; b < a.row_blocks; ++b) total += a.partial[b * a.channels * (W + 1) + i];
    const int64_t c = i / (W + 1), k = i % (W + 1);
    if (k < W) a.dweight[c * W + k] = total;
    else if (a.dbias) a.dbias[c] = total;
}

// ===========================================================================
// selective scan:  d = softplus(delta + bias),  h = exp(d A) h + d x B,  y = (C h + skip x) silu(z)
// LN neighbouring lanes share a channel, four states each.
// ===========================================================================
template <class T>
__device__ __forceinline__ void load_states(const T* p, int first, int n, float (&v)[kStates]) {
#pragma unroll
    for (int i = 0; i < kStates; ++i) v[i] = first + i < n ? load1(p + first + i) : 0.0f;
}

template <int LN>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
    for (int m = 1; m < LN; m *= 2) v += __shfl_xor_sync(kFull, v, m);
    return v;
}

// four elements as stored
template <class T> struct Raw4 { T e[4]; };
template <class T>
__device__ __forceinline__ void put4(T* p, bool vec, int n, const float (&v)[4]) {
    if (vec && n == 4) {
        Raw4<T> r;
#pragma unroll
        for (int i = 0; i < 4; ++i) store1(&r.e[i], v[i]);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.e);
        else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(r.e);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < n) store1(p + i, v[i]);
    }
}

// To shared memory: asynchronous where it is one aligned access of a whole vector; the first n, zeros for the rest.
template <class T>
__device__ __forceinline__ void copy4(T* to, const T* from, bool vec, int n) {
    if (vec && n == 4) {
        const unsigned at = (unsigned)__cvta_generic_to_shared(to);
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(4 * sizeof(T)) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = i < n ? from[i] : T(0.0f);
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT = 0>     // groups that may still be under way
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
template <class T>
__device__ __forceinline__ Raw4<T> raw4(const T* p) {       // from shared memory, aligned to four elements
    Raw4<T> r;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(r.e) = *reinterpret_cast<const uint4*>(p);
    else *reinterpret_cast<uint2*>(r.e) = *reinterpret_cast<const uint2*>(p);
    return r;
}

// exp(d A) for a rate as scan_rate() prepares it: FAST folds log2(e) into the rate.  An infinite rate becomes
// the largest finite one, whose decay over any step is the same, so that a tile's tokens behind the
// sequence's end (steps of length zero) leave the state as it is instead of multiplying zero by infinity.
__device__ __forceinline__ float scan_rate(float A) {
#if PD_MODE == 2
    A *= 1.4426950408889634f;
#endif
    return fabsf(A) == INFINITY ? copysignf(3.4028234e38f, A) : A;
}
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float decay(float d, float rate) {
#if PD_MODE == 2
    return exp2_approx(d * rate);
#else
    return expf(d * rate);
#endif
}
__device__ __forceinline__ pair_t decay2(pair_t d, pair_t rate) {
    float x, y;
    unpack(mul2(d, rate), x, y);
#if PD_MODE == 2
    return pack(exp2_approx(x), exp2_approx(y));
#else
    return pack(expf(x), expf(y));
#endif
}

// The same where a decay's own error matters: in the gradients, whose sums over thousands of tokens carry it along, in
// single steps, whose state comes back thousands of times, and in prompts of float32 tokens.  Near one, where a state
// remembers for long, the approximate power's 2^-22 is four times a rounding.  There, |d A log2(e)| < 0.1, the series of
// 2^v to the fourth power takes its place; it ends 1.3e-8 short of the sum.  (Decays around 1 - 1e-2, 4096 tokens, error
// of the last state: 1.4e-6 with the approximate power, 2.1e-7 with the series, 2.9e-7 in SAFE; fed back step by step
// 2.8e-6, 2.6e-7, 4.3e-7.  It takes a float32 prompt of 4 x 2048 x 2048 x 16 from 194 to 223 us, one of 32 x 512 x 4096
// x 16, which fills the GPU, from 680 to 911; 2-byte tokens, whose inputs are 2^-9 off, keep the approximate power: the
// series would take the first from 186 to 221 us.)
constexpr float kPower1 = 0.6931471805599453f, kPower2 = 0.2402265069591007f, kPower3 = 0.0555041086648216f,
                kPower4 = 0.0096181291076285f;
__device__ __forceinline__ pair_t decay2_fine(pair_t d, pair_t rate) {
#if PD_MODE == 2
    const pair_t v = mul2(d, rate);
    pair_t p = mad2(pack(kPower4, kPower4), v, pack(kPower3, kPower3));
    p = mad2(p, v, pack(kPower2, kPower2));
    p = mad2(p, v, pack(kPower1, kPower1));
    p = mad2(p, v, pack(1.0f, 1.0f));
    float x, y, px, py;
    unpack(v, x, y);
    unpack(p, px, py);
    return pack(fabsf(x) < 0.1f ? px : exp2_approx(x), fabsf(y) < 0.1f ? py : exp2_approx(y));
#else
    return decay2(d, rate);
#endif
}
__device__ __forceinline__ float decay_fine(float d, float rate) {
#if PD_MODE == 2
    const float v = d * rate;
    const float p = fmaf(fmaf(fmaf(fmaf(kPower4, v, kPower3), v, kPower2), v, kPower1), v, 1.0f);
    return fabsf(v) < 0.1f ? p : exp2_approx(v);
#else
    return decay(d, rate);
#endif
}

// exp(total A) v over many tokens at once.  The factor may leave float32's range where the product does not (a state
// of zero, or a small one, that grows): it is then taken as two halves, and a state of zero stays zero.
__device__ __forceinline__ float carried(float v, float total, float rate) {
    const float whole = decay_fine(total, rate);
    if (whole >= 1.1754944e-38f && whole <= 3.4028234e38f) return whole * v;
    const float half = decay(0.5f * total, rate);
    return v == 0.0f ? 0.0f : half * (half * v);
}

// One token per sequence; state in and out may be the same memory.  Bound: the states, read and written once, 8
// bytes per state: LN neighbouring lanes read a channel's states as one 16-byte vector each (VEC), a warp 512 bytes.
template <class T, int LN, bool VEC>
__global__ void __launch_bounds__(256) pd_selective_scan_step_kernel(PdScanArgs a) {
    // blockIdx.x and the warps across channels, blockIdx.y across sequences: a thread works for one token, and a
    // division for its place would cost it more than the rest (49 us for 256 x 4096 x 16 with four of them; 43 with one
    // sequence per thread, two thirds of whose instructions were addresses)
    const int per = (int)(a.channels / a.groups), ch = 32 / LN, tiles = (per + ch - 1) / ch;
    const int job = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, group = a.groups == 1 ? 0 : job / tiles;
    if (group >= a.groups || (a.groups == 1 && job >= tiles)) return;
    const int lane = threadIdx.x & 31, sub = lane % LN, first = sub * kStates;
    const int within = (job - group * tiles) * ch + lane / LN;
    const bool active = within < per;
    const int64_t c = group * per + (active ? within : per - 1);     // an idle lane repeats the last channel
    float A[kStates];
    if (VEC) {
        const float4 q = *reinterpret_cast<const float4*>(a.A + c * a.state + first);
        A[0] = q.x; A[1] = q.y; A[2] = q.z; A[3] = q.w;
    } else {
        load_states(a.A + c * a.state, first, a.state, A);
    }
#pragma unroll
    for (int i = 0; i < kStates; ++i) A[i] = scan_rate(A[i]);
    const float bias = a.bias ? a.bias[c] : 0.0f, skip = a.skip ? a.skip[c] : 0.0f;
    // a block takes `run` sequences one after another, the next one's operands on their way
    const int64_t s0 = (int64_t)blockIdx.y * a.run;
    const int left = (int)(a.tok.seqs - s0 < a.run ? a.tok.seqs - s0 : a.run);
    const int64_t step = a.channels, step_h = a.channels * a.state, step_bc = (int64_t)a.groups * a.state;
    const T* px = (const T*)a.x + s0 * step + c;
    const T* pd = (const T*)a.delta + s0 * step + c;
    const T* pz = a.z ? (const T*)a.z + s0 * step + c : nullptr;
    const T* pB = (const T*)a.B + s0 * step_bc + group * a.state;
    const T* pC = (const T*)a.C + s0 * step_bc + group * a.state;
    const float* ph = a.initial + s0 * step_h + c * a.state;
    T* py = (T*)a.y + s0 * step + c;
    float* po = a.final_state + s0 * step_h + c * a.state;
    struct Operands { float h[kStates], B[kStates], C[kStates], x, d, z; };
    auto fetch_next = [&](Operands& q) {
        if (VEC) {
            const float4 v = *reinterpret_cast<const float4*>(ph + first);
            q.h[0] = v.x; q.h[1] = v.y; q.h[2] = v.z; q.h[3] = v.w;
            load<4>(pB + first, q.B);
            load<4>(pC + first, q.C);
        } else {
            load_states(ph, first, a.state, q.h);
            load_states(pB, first, a.state, q.B);
            load_states(pC, first, a.state, q.C);
        }
        q.x = load1(px);
        q.d = load1(pd);
        q.z = pz ? load1(pz) : 0.0f;
        ph += step_h; pB += step_bc; pC += step_bc; px += step; pd += step;
        if (pz) pz += step;
    };
    Operands now, next;
    fetch_next(now);
    for (int k = 0; k < left; ++k) {
        if (k + 1 < left) fetch_next(next);
        float d = now.d + bias;
        if (a.softplus) d = softplus_(d);
        const float u = d * now.x;
        float h[kStates], y = 0.0f;
#pragma unroll
        for (int i = 0; i < kStates; ++i) {
            const bool in = VEC || first + i < a.state;
            h[i] = decay_fine(d, A[i]) * now.h[i] + (in ? u * now.B[i] : 0.0f);
            y += in ? now.C[i] * h[i] : 0.0f;
        }
        y = sum_lanes<LN>(y);
        if (a.skip) y += skip * now.x;
        if (a.z) y *= now.z * sigmoid_(now.z);
        if (active) {
            if (sub == 0) store1(py, y);
            if (VEC) {
                *reinterpret_cast<float4*>(po + first) = make_float4(h[0], h[1], h[2], h[3]);
            } else {
#pragma unroll
                for (int i = 0; i < kStates; ++i) if (first + i < a.state) po[first + i] = h[i];
            }
        }
        py += step;
        po += step_h;
        now = next;
    }
}

// ---------------------------------------------------------------------------
// what the prompt and gradient kernels share
// ---------------------------------------------------------------------------
__device__ __forceinline__ pair_t shift_up(pair_t v, int by) {
    float x, y;
    unpack(v, x, y);
    return pack(__shfl_up_sync(kFull, x, by), __shfl_up_sync(kFull, y, by));
}
__device__ __forceinline__ pair_t shift_down(pair_t v, int by) {
    float x, y;
    unpack(v, x, y);
    return pack(__shfl_down_sync(kFull, x, by), __shfl_down_sync(kFull, y, by));
}
__device__ __forceinline__ pair_t from_lane(pair_t v, int lane) {
    float x, y;
    unpack(v, x, y);
    return pack(__shfl_sync(kFull, x, lane), __shfl_sync(kFull, y, lane));
}
// Whether products of the decays `up` of up to TL / 2 token groups stay finite, for all of a warp (decays of negative
// rates are at most one): an infinite one would turn a state of zero into NaN.
template <int TL>
__device__ __forceinline__ bool within_range(const pair_t (&up)[2]) {
    constexpr float most = TL == 8 ? 2147483648.0f : TL == 16 ? 32768.0f : 128.0f;      // 2^(126 / (TL / 2)) or less
    static_assert(TL == 8 || TL == 16 || TL == 32, "");
    float a, b, c, d;
    unpack(up[0], a, b);
    unpack(up[1], c, d);
    return __all_sync(kFull, a <= most && b <= most && c <= most && d <= most);
}
// v[i] summed over the K lanes of a group, lane i keeping the i-th sum
template <int K>
__device__ __forceinline__ float sum_to_lane(const float (&v)[K], int sub) {
    if constexpr (K == 1) {
        return v[0];
    } else if constexpr (K == 2) {
        return (sub & 1 ? v[1] : v[0]) + __shfl_xor_sync(kFull, sub & 1 ? v[0] : v[1], 1);
    } else {
        const float lo = (sub & 1 ? v[1] : v[0]) + __shfl_xor_sync(kFull, sub & 1 ? v[0] : v[1], 1);
        const float hi = (sub & 1 ? v[3] : v[2]) + __shfl_xor_sync(kFull, sub & 1 ? v[2] : v[3], 1);
        return (sub & 2 ? hi : lo) + __shfl_xor_sync(kFull, sub & 2 ? lo : hi, 2);
    }
}
// a pair of states of which the first n exist
__device__ __forceinline__ pair_t keep_states(pair_t v, int n) {
    float x, y;
    unpack(v, x, y);
    return pack(n > 0 ? x : 0.0f, n > 1 ? y : 0.0f);
}
template <int K>
__device__ __forceinline__ void load_pairs(const float2* p, pair_t (&v)[K]) {
    if constexpr (K == 1) {
        v[0] = *reinterpret_cast<const pair_t*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < K; i += 2) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(p + i);
            v[i] = q.x;
            v[i + 1] = q.y;
        }
    }
}

// ---------------------------------------------------------------------------
// The prompt kernel.  A lane holds four states of NCH neighbouring channels and walks the tokens one by one; LN
// lanes share a channel, 32 / LN * NCH channels make a warp's.  Two of a block's four warps walk; the other two bring
// tiles of 32 tokens to shared memory as float32 (step lengths, inputs, couplings) ahead of them, the elements of the
// tile after on their way, and finish the outputs behind them (skip, gate, rounding), with one barrier per tile.
//
// Bound: the exponentials, one per (token, channel, state), 16 per clock and SM: 8 cycles per warp instruction and
// scheduler.  Beside each stand 2 packed multiply-adds and, with two channels per lane, 1.75 words of shared memory
// (7 of the 8 cycles).  4 x 2048 tokens x 2048 channels x 16 states in bf16 take 178 us, 58 of them what the
// exponentials cannot do without: 512 blocks are 1.7 walking warps per scheduler, too few to hide what each waits
// for (212 us with staging and walking in turn by the same two warps; five blocks of 96 registers on an SM
// instead of four of 120 take 3 % more here and 8 % less where a sequence is cut).  Forms that hold tokens across lanes or warps
// instead, so as to fill the GPU with one sequence, needed 18 to 31 instructions per state for their scans (8192 x
// 2048 x 16 took 417 us); so a call with few sequences and channels is cut into segments of tokens: a first launch
// (STATE) takes each from a zero state to its end state and total step, and the blocks of the second compose the state
// entering theirs.
// ---------------------------------------------------------------------------
constexpr int kStageThreads = 64, kScanThreads = 32 * PD_SCAN_WALKING_WARPS + kStageThreads;

// all of the block's warps, which reach it from different places
__device__ __forceinline__ void tile_barrier() { asm volatile("barrier.sync 1, %0;" ::"n"(kScanThreads) : "memory"); }

// segments: where a sequence's first one is counted, and the sequence of the id-th (an empty one has one, too)
__device__ __forceinline__ int64_t dense_segments(const PdScanArgs& a) {
    return a.tok.length > a.segment ? (a.tok.length + a.segment - 1) / a.segment : 1;
}
__device__ __forceinline__ int64_t first_segment(const PdScanArgs& a, int64_t s, int64_t begin) {
    return a.tok.offsets ? begin / a.segment + s : s * dense_segments(a);
}
__device__ __forceinline__ int64_t segment_owner(const PdScanArgs& a, int64_t id) {
    if (!a.tok.offsets) return id / dense_segments(a);
    int64_t lo = 0, hi = a.tok.seqs;    // the last s whose first segment is not behind id
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (first_segment(a, mid, clamp_row(a.tok.offsets[mid], a.tok.rows)) <= id) lo = mid + 1; else hi = mid;
    }
    return lo - 1;
}

template <class T, int LN, int NCH, bool FULL, bool STATE>
__global__ void __launch_bounds__(kScanThreads, PdScanShape(LN, NCH, sizeof(T)).resident()) pd_selective_scan_kernel(PdScanArgs a) {
    constexpr PdScanShape G(LN, NCH, sizeof(T));
    constexpr int kRow = G.kRow, quads = G.channels / 4, kPass = kStageThreads / quads;
    static_assert(kStageThreads % quads == 0 && kRow % kPass == 0 && G.warp_channels % 4 == 0, "staging covers a tile");
    extern __shared__ float4 smem4[];
    float* smem = reinterpret_cast<float*>(smem4);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % LN, cl = lane / LN, first = sub * 4;
    const int64_t per = a.channels / a.groups, tiles = (per + G.channels - 1) / G.channels, all = tiles * a.groups;
    const int64_t id = blockIdx.x / all, tile = blockIdx.x - id * all;
    const int64_t group = a.groups == 1 ? 0 : tile / tiles, within = (tile - group * tiles) * G.channels;
    const int64_t c0 = group * per + within;                            // the block's first channel
    const int count = (int)(per - within < G.channels ? per - within : G.channels);
    if (id >= a.segments) {     // (packed calls: a few more)
        clear_free_rows(a.tok, a.channels, (T*)a.y, (id - a.segments) * all + tile, a.free_blocks * all);
        return;
    }
    const int64_t s = segment_owner(a, id);
    if (s < 0) return;
    int64_t begin, end;
    bounds_of(a.tok, s, begin, end);
    const int64_t id0 = first_segment(a, s, begin), number = id - id0;
    const int64_t start = begin + number * a.segment, stop = start + a.segment < end ? start + a.segment : end;
    if (number < 0 || (number > 0 && start >= end)) return;
    if (STATE && stop == end) return;         // nothing follows a last segment
    const bool computes = warp < PD_SCAN_WALKING_WARPS;
    // this lane's channels, their rates and the state entering
    pair_t rate[NCH][2], h[NCH][2];
    const int mine = warp * G.warp_channels + cl * NCH;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        const bool in = computes && mine + j < count;
        const int64_t c = c0 + (in ? mine + j : 0);
        float A[4], v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        load_states(a.A + c * a.state, first, a.state, A);
#pragma unroll
        for (int i = 0; i < 4; ++i) A[i] = scan_rate(A[i]);
        if (!STATE && computes) {
            if (a.initial) load_states(a.initial + (s * a.channels + c) * a.state, first, a.state, v);
            for (int64_t k = id0; k < id; ++k) {
                const float total = a.totals[k * a.channels + c];
                float e[4];
                load_states(a.ends + (k * a.channels + c) * a.state, first, a.state, e);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = carried(v[i], total, A[i]) + e[i];
            }
        }
        rate[j][0] = pack(A[0], A[1]);
        rate[j][1] = pack(A[2], A[3]);
        h[j][0] = pack(v[0], v[1]);
        h[j][1] = pack(v[2], v[3]);
    }
    auto keep = [&](float* to, int j) {        // the states of channel j
        float v[4];
        unpack(h[j][0], v[0], v[1]);
        unpack(h[j][1], v[2], v[3]);
        if (mine + j >= count) return;
        to += (c0 + mine + j) * a.state + first;
        if (FULL && a.vec_params) {
            *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (first + i < a.state) to[i] = v[i];
        }
    };
    // staging: four channels of a token per thread, always the same channels
    const int stid = tid & (kStageThreads - 1), c4 = stid % quads * 4, st = stid / quads;
    const int left = count - c4 < 0 ? 0 : count - c4 > 4 ? 4 : count - c4;
    float bias[4], skip[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = a.bias && i < left ? a.bias[c0 + c4 + i] : 0.0f;
        skip[i] = a.skip && i < left ? a.skip[c0 + c4 + i] : 0.0f;
    }
    const int64_t chunk0 = first_chunk(a.tok, s, begin), stride = (int64_t)a.groups * a.state;
    T* raw = reinterpret_cast<T*>(reinterpret_cast<char*>(smem) + G.raw);
    T* couplings = raw + 12 * kRow * G.channels;
    constexpr int cells = kRow * G.channels;
    const bool gate = !STATE && a.z;
    const int tiles_here = (int)((stop - start + kRow - 1) / kRow);
    auto copy_tile = [&](int k) {
        const int64_t from = start + (int64_t)k * kRow;
        if (k >= tiles_here) { copies_commit(); return; }      // (each tile one group, for the wait to count)
        T* to = raw + (k & 3) * 3 * cells + st * G.channels + c4;
        T* to_bc = couplings + (k & 1) * 2 * kRow * G.pad;
        int64_t at = (from + st) * a.channels + c0 + c4;
#pragma unroll 2
        for (int t = st; t < kRow; t += kPass) {
            const int n = from + t < stop ? left : 0;
            copy4(to, (const T*)a.x + at, a.vec, n);
            copy4(to + cells, (const T*)a.delta + at, a.vec, n);
            if (gate) copy4(to + 2 * cells, (const T*)a.z + at, a.vec, n);
            to += kPass * G.channels;
            at += kPass * a.channels;
        }
#pragma unroll 2
        for (int i = stid; i < kRow * LN; i += kStageThreads) {
            const int t = i / LN, n4 = i % LN * 4;
            int n = from + t < stop ? a.state - n4 : 0;
            n = n < 0 ? 0 : n > 4 ? 4 : n;
            const int64_t at = (from + t) * stride + group * a.state + n4;
            copy4(to_bc + 4 * i, (const T*)a.B + at, a.vec_states, n);
            if (!STATE) copy4(to_bc + kRow * G.pad + 4 * i, (const T*)a.C + at, a.vec_states, n);
        }
        copies_commit();
    };
    // a tile's elements to float32 (each thread reads back what it has fetched itself)
    auto stage = [&](int k) {
        const int tokens = (int)(stop - start - (int64_t)k * kRow < kRow ? stop - start - (int64_t)k * kRow : kRow);
        const T* got = raw + (k & 3) * 3 * cells + st * G.channels + c4;
        float* du = smem + G.du + (k & 1) * 2 * cells;
        for (int t = st; t < kRow; t += kPass, got += kPass * G.channels) {
            const Raw4<T> rx = raw4(got), rd = raw4(got + cells);
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float d = load1(&rd.e[i]) + bias[i];
                if (a.softplus) d = softplus_(d);
                d = t < tokens ? d : 0.0f;
                v[i] = make_float2(d, d * load1(&rx.e[i]));
            }
            // (every other four threads store their second half first: no two of eight meet in a bank)
            float4* to = reinterpret_cast<float4*>(du + 2 * (t * G.channels + c4));
            const float4 low = make_float4(v[0].x, v[0].y, v[1].x, v[1].y), high = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
            const int turn = lane >> 2 & 1;
            to[turn] = turn ? high : low;
            to[turn ^ 1] = turn ? low : high;
        }
        const T* bc = couplings + (k & 1) * 2 * kRow * G.pad;
        for (int i = stid; i < kRow * LN; i += kStageThreads) {
            const Raw4<T> b = raw4(bc + 4 * i);
            reinterpret_cast<float4*>(smem + G.B + (k & 1) * kRow * G.pad)[i] =
                make_float4(load1(&b.e[0]), load1(&b.e[1]), load1(&b.e[2]), load1(&b.e[3]));
            if (!STATE) {
                const Raw4<T> c = raw4(bc + kRow * G.pad + 4 * i);
                reinterpret_cast<float4*>(smem + G.C + (k & 1) * kRow * G.pad)[i] =
                    make_float4(load1(&c.e[0]), load1(&c.e[1]), load1(&c.e[2]), load1(&c.e[3]));
            }
        }
    };
    // a tile's outputs: the sums, the skip and the gate
    auto finish = [&](int k) {
        const int64_t from = start + (int64_t)k * kRow;
        const int tokens = (int)(stop - from < kRow ? stop - from : kRow);
        const T* got = raw + (k & 3) * 3 * cells + st * G.channels + c4;
        const float* sum = smem + G.y + (k & 1) * cells + c4 / G.warp_channels * kRow * G.warp_channels + c4 % G.warp_channels;
        T* to = (T*)a.y + (from + st) * a.channels + c0 + c4;
        for (int t = st; t < tokens; t += kPass, got += kPass * G.channels, to += kPass * a.channels) {
            const Raw4<T> rx = raw4(got);
            const float4 q = *reinterpret_cast<const float4*>(sum + t * G.warp_channels);
            float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += skip[i] * load1(&rx.e[i]);
            if (gate) {
                const Raw4<T> rz = raw4(got + 2 * cells);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float z = load1(&rz.e[i]);
                    v[i] *= z * sigmoid_(z);
                }
            }
            put4(to, a.vec, left, v);
        }
    };
    float total[NCH] = {};
    if (!computes && tiles_here > 0) {
        copy_tile(0);
        copy_tile(1);
        copies_wait<1>();
        stage(0);
    }
    tile_barrier();
    // One barrier per tile: while two warps walk tile k, the other two finish tile k - 1 and stage tile k + 1, with
    // tile k + 2 on its way.
    for (int k = 0; k < tiles_here; ++k) {
        const int64_t from = start + (int64_t)k * kRow;
        if (!computes) {
            if (!STATE && k > 0) finish(k - 1);
            if (k + 1 < tiles_here) {
                copy_tile(k + 2);
                copies_wait<1>();
                stage(k + 1);
            }
            tile_barrier();
            continue;
        }
        if (!STATE && a.carries) {
            float* to = a.carries + (chunk0 + (from - begin) / PD_SCAN_CHUNK) * a.channels * a.state;
#pragma unroll
            for (int j = 0; j < NCH; ++j) keep(to, j);
        }
        const float* du = smem + G.du + (k & 1) * 2 * cells + 2 * mine;
        const float* tile_B = smem + G.B + (k & 1) * kRow * G.pad + first;
        const float* tile_C = smem + G.C + (k & 1) * kRow * G.pad + first;
        float* out = smem + G.y + (k & 1) * cells + warp * kRow * G.warp_channels + cl * NCH;     // (warp, token, channel)
        float sums[NCH] = {};
        // Four tokens at a time: their operands are read before the outputs of the four before them are stored (the
        // compiler would not move a read of shared memory past a store to it), so that sixteen exponentials are
        // under way at once.
        constexpr int F = 4;
        struct Operands { float d[F][NCH], u[F][NCH]; ulonglong2 B[F], C[F]; };
        auto fetch_tokens = [&](int t, Operands& q) {
#pragma unroll
            for (int i = 0; i < F; ++i) {
                if constexpr (NCH == 2) {
                    const float4 v = *reinterpret_cast<const float4*>(du + 2 * (t + i) * G.channels);
                    q.d[i][0] = v.x; q.u[i][0] = v.y; q.d[i][NCH - 1] = v.z; q.u[i][NCH - 1] = v.w;
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(du + 2 * (t + i) * G.channels);
                    q.d[i][0] = v.x; q.u[i][0] = v.y;
                }
                q.B[i] = *reinterpret_cast<const ulonglong2*>(tile_B + (t + i) * G.pad);
                if (!STATE) q.C[i] = *reinterpret_cast<const ulonglong2*>(tile_C + (t + i) * G.pad);
            }
        };
        Operands q;
        fetch_tokens(0, q);
#pragma unroll 2
        for (int t = 0; t < kRow; t += F) {
            // (tokens behind the segment's end have steps and inputs of zero)
            pair_t w[F][NCH][2], b[F][NCH][2];
            float y[F][NCH];
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const pair_t step = pack(q.d[i][j], q.d[i][j]), in = pack(q.u[i][j], q.u[i][j]);
                    w[i][j][0] = sizeof(T) == 4 ? decay2_fine(step, rate[j][0]) : decay2(step, rate[j][0]);
                    w[i][j][1] = sizeof(T) == 4 ? decay2_fine(step, rate[j][1]) : decay2(step, rate[j][1]);
                    b[i][j][0] = mul2(in, q.B[i].x);
                    b[i][j][1] = mul2(in, q.B[i].y);
                    if (!FULL) {     // states beyond the last one stay zero whatever the input is
                        b[i][j][0] = keep_states(b[i][j][0], a.state - first);
                        b[i][j][1] = keep_states(b[i][j][1], a.state - first - 2);
                    }
                    if (STATE) sums[j] += q.d[i][j];
                }
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    h[j][0] = mad2(w[i][j][0], h[j][0], b[i][j][0]);
                    h[j][1] = mad2(w[i][j][1], h[j][1], b[i][j][1]);
                    if (!STATE) y[i][j] = halves(mad2(q.C[i].y, h[j][1], mul2(q.C[i].x, h[j][0])));
                }
            if (t + F < kRow) fetch_tokens(t + F, q);
            if (!STATE)
#pragma unroll
                for (int i = 0; i < F; i += (LN < 4 ? LN : 4)) {
                    // an output's sum over its lanes; lane k keeps the k-th of LN (at most four) tokens
                    float v[NCH];
#pragma unroll
                    for (int j = 0; j < NCH; ++j) {
                        constexpr int K = LN < 4 ? LN : 4;
                        float part[K];
#pragma unroll
                        for (int k = 0; k < K; ++k) part[k] = y[i + k][j];
                        v[j] = sum_to_lane<K>(part, sub);
#pragma unroll
                        for (int m = 4; m < LN; m *= 2) v[j] += __shfl_xor_sync(kFull, v[j], m);
                    }
                    if (LN <= 4 || sub < 4) {
                        float* to = out + (t + i + (LN > 1 ? sub : 0)) * G.warp_channels;
                        if constexpr (NCH == 2) *reinterpret_cast<float2*>(to) = make_float2(v[0], v[NCH - 1]);
                        else to[0] = v[0];
                    }
                }
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) total[j] += sums[j];
        tile_barrier();
    }
    if (!computes) {
        if (!STATE && tiles_here > 0) finish(tiles_here - 1);
        return;
    }
    if (STATE) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            keep(a.ends + id * a.channels * a.state, j);
            if (sub == 0 && mine + j < count) a.totals[id * a.channels + c0 + mine + j] = total[j];
        }
    } else if (a.final_state && stop == end) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) keep(a.final_state + s * a.channels * a.state, j);
    }
}

// ---------------------------------------------------------------------------
// Gradients, chunk by chunk of 32 tokens from the end.  A block owns four warps' channels of one group and one
// sequence.  A warp takes its channels one after another, each over the whole chunk at once: a lane holds K
// tokens' four states, LN lanes the states of a token group, 32 / LN lanes the token groups.  Forward from the
// state kept at the chunk's start, then backwards,
//     g_t = C_t dy_t + a_{t+1} g_{t+1},   dA += d a h_{t-1} g,  ddelta: A a h_{t-1} g + x B g,  dB += u g,  dC += dy h,
// both as a pass from zero, a scan over the token groups by shuffles and a second pass from the true value.
// Tokens stand across lanes, so the sums of dB and dC over channels, shared by the whole group, stay in registers
// while a warp goes through its channels; only their sum over the four warps passes through shared memory.
// LN == K, and after the sums over a token's LN lanes each lane finishes one token.
//
// Bound: instruction issue.  4 x 2048 tokens x 2048 channels x 16 states in bf16 take 640 us: 41 instructions per
// state at 0.53 a clock and scheduler with three blocks of 168 registers on an SM (eight warps of 128 registers a block spilled, 1120 us; operands read where they are used
// instead of a chunk ahead, 1030 us).
// ---------------------------------------------------------------------------
constexpr int kGradThreads = 32 * PD_SCAN_GRAD_WARPS;

template <class T, int LN, bool GATE, bool ONE>
__global__ void __launch_bounds__(kGradThreads, 3) pd_selective_scan_grad_kernel(PdScanArgs a) {
    constexpr int K = LN, TL = 32 / LN, kRow = PD_SCAN_CHUNK, kWide = 4 * LN;
    static_assert(K * TL == kRow, "a warp covers a chunk");
    extern __shared__ float4 smem4[];
    float* smem = reinterpret_cast<float*>(smem4);
    const PdGradShape<LN, ONE> G(a.state, a.per_warp, sizeof(T));
    float *sX = smem + G.x, *sS = smem + G.s, *sZ = smem + G.z;
    float2 *sD = reinterpret_cast<float2*>(smem + G.d), *sU = reinterpret_cast<float2*>(smem + G.u), *sG = reinterpret_cast<float2*>(smem + G.g);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % LN, tl = lane / LN;
    const int64_t per = a.channels / a.groups, tiles = (per + G.channels - 1) / G.channels;
    const int64_t job = blockIdx.x, s = job / (tiles * a.groups);
    const int64_t group = job / tiles % a.groups, within = job % tiles * G.channels;
    const int64_t c0 = group * per + within;
    const int count = (int)(per - within < G.channels ? per - within : G.channels);
    float* bc_out = a.partial_bc + job % (tiles * a.groups) * a.tok.rows * 2 * G.pad;
    int64_t begin, end;
    bounds_of(a.tok, s, begin, end);
    // swizzled places of (channel, token): four channels of a token and four tokens of a channel are both
    // reached without bank conflicts
    auto place = [](int c, int t) { return c * kRow + (t ^ ((c >> 2 & 7) << 2)); };
    for (int i = tid; i < G.channels * G.pad; i += kGradThreads) {
        const int c = i / G.pad, n = i % G.pad;
        smem[G.carry + i] = a.dfinal && c < count && n < a.state ? a.dfinal[(s * a.channels + c0 + c) * a.state + n] : 0.0f;
    }
    for (int i = tid; i < G.channels * G.pad; i += kGradThreads) {
        const int c = i / G.pad, n = i % G.pad;
        smem[G.rate + i] = c < count && n < a.state ? scan_rate(a.A[(c0 + c) * a.state + n]) : 0.0f;
    }
    for (int i = tid; i < G.channels * G.slices * 128; i += kGradThreads) smem[G.dA + i] = 0.0f;
    if (tid < G.channels) smem[G.skip + tid] = a.skip && tid < count ? a.skip[c0 + tid] : 0.0f;
    // staging: four channels of a token per thread, always the same channels
    const int quads = G.channels / 4, rows = kGradThreads / quads, c4 = tid % quads * 4;
    const bool stages = tid < rows * quads;     // (128 threads need not divide into rows: the last ones rest)
    const int st = stages ? tid / quads : kRow;
    const int left = count - c4 < 0 ? 0 : count - c4 > 4 ? 4 : count - c4;
    float bias[4], dbias[4], dskip[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = a.bias && i < left ? a.bias[c0 + c4 + i] : 0.0f;
        dbias[i] = dskip[i] = 0.0f;
    }
    const int64_t chunks = (end - begin + kRow - 1) / kRow, chunk0 = first_chunk(a.tok, s, begin);
    const int64_t stride = (int64_t)a.groups * a.state;
    T* raw = reinterpret_cast<T*>(reinterpret_cast<char*>(smem) + G.raw);
    T* couplings = reinterpret_cast<T*>(reinterpret_cast<char*>(smem) + G.couplings);
    const int cells = kRow * G.channels;
    // a chunk's operands on their way while the one behind it is worked on
    auto copy_chunk = [&](int64_t k) {
        const int64_t from = begin + k * kRow;
        for (int t = st; t < kRow; t += rows) {
            const int n = from + t < end ? left : 0, to = t * G.channels + c4;
            const int64_t at = (from + t) * a.channels + c0 + c4;
            copy4(raw + to, (const T*)a.x + at, a.vec, n);
            copy4(raw + cells + to, (const T*)a.delta + at, a.vec, n);
            copy4(raw + 2 * cells + to, (const T*)a.dy + at, a.vec, n);
            if (GATE) copy4(raw + 3 * cells + to, (const T*)a.z + at, a.vec, n);
        }
        for (int i = tid; i < kRow * (G.pad / 4); i += kGradThreads) {
            const int t = i / (G.pad / 4), n4 = i % (G.pad / 4) * 4;
            int n = from + t < end ? a.state - n4 : 0;
            n = n < 0 ? 0 : n > 4 ? 4 : n;
            const int64_t at = (from + t) * stride + group * a.state + n4;
            T* to = couplings + ((int)(k & 1) * 2 * kRow + t) * G.pitch + n4;
            copy4(to, (const T*)a.B + at, a.vec_states, n);
            copy4(to + kRow * G.pitch, (const T*)a.C + at, a.vec_states, n);
        }
        for (int i = tid; i < G.channels * (G.pad / 4); i += kGradThreads) {
            const int c = i / (G.pad / 4), n4 = i % (G.pad / 4) * 4;
            int n = c < count ? a.state - n4 : 0;
            n = n < 0 ? 0 : n > 4 ? 4 : n;
            copy4(smem + G.entry + ((int)(k & 1) * G.channels + c) * G.pad + n4,
                  a.carries_in + ((chunk0 + k) * a.channels + c0 + c) * a.state + n4, a.vec_params, n);
        }
        copies_commit();
    };
    if (chunks > 0) copy_chunk(chunks - 1);
    for (int64_t k = chunks - 1; k >= 0; --k) {
        const int64_t from = begin + k * kRow;
        copies_wait();
        // (each thread reads back what it has fetched itself)
        for (int t = st; t < kRow; t += rows) {
            const int n = from + t < end ? left : 0, to = t * G.channels + c4;
            const Raw4<T> rx = raw4(raw + to), rd = raw4(raw + cells + to), rg = raw4(raw + 2 * cells + to);
            Raw4<T> rz;
            if (GATE) rz = raw4(raw + 3 * cells + to);
            const int row = place(c4, t);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = row + i * kRow;
                const float x = load1(&rx.e[i]), bent = load1(&rd.e[i]) + bias[i];
                float d = bent, slope = 1.0f, g = load1(&rg.e[i]);
                if (a.softplus) d = softplus_(bent, slope);
                if (GATE) {
                    const float z = load1(&rz.e[i]), sig = sigmoid_(z);
                    sZ[at] = g * (sig * (1.0f + z * (1.0f - sig)));
                    g *= z * sig;
                }
                // (what lies behind the sequence's end was fetched as zeros)
                d = i < n ? d : 0.0f;
                sX[at] = x;
                sD[at] = make_float2(d, d);
                sU[at] = make_float2(d * x, d * x);
                sG[at] = make_float2(g, g);
                sS[at] = slope;
                dskip[i] += g * x;
            }
        }
        if (k > 0) copy_chunk(k - 1);
        __syncthreads();
        for (int q = 0; q < G.slices; ++q) {
            const int first = q * kWide + sub * 4;
            pair_t B[K][2], C[K][2], dB[K][2], dC[K][2];
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const T* from_row = couplings + ((int)(k & 1) * 2 * kRow + tl * K + i) * G.pitch + first;
                const Raw4<T> b = raw4(from_row), c = raw4(from_row + kRow * G.pitch);
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    B[i][p] = pack(load1(&b.e[2 * p]), load1(&b.e[2 * p + 1]));
                    C[i][p] = pack(load1(&c.e[2 * p]), load1(&c.e[2 * p + 1]));
                    dB[i][p] = dC[i][p] = pack(0.0f, 0.0f);
                }
            }
            for (int cc = 0; cc < a.per_warp; ++cc) {
                const int c = warp * a.per_warp + cc;
                if (c >= count) break;
                pair_t rate[2], entry[2], leave[2];
                const pair_t* rates = reinterpret_cast<const pair_t*>(smem + G.rate + c * G.pad + first);
                const pair_t* entries = reinterpret_cast<const pair_t*>(smem + G.entry + ((int)(k & 1) * G.channels + c) * G.pad + first);
                rate[0] = rates[0];
                rate[1] = rates[1];
                entry[0] = entries[0];
                entry[1] = entries[1];
                float* kept = smem + G.carry + c * G.pad + first;
                leave[0] = *reinterpret_cast<const pair_t*>(kept);
                leave[1] = *reinterpret_cast<const pair_t*>(kept + 2);
                float y[K], du[K], dd[K];
                const int here = place(c, tl * K);
                pair_t u[K], gg[K];
                load_pairs<K>(sU + here, u);
                load_pairs<K>(sG + here, gg);
                // both directions from zero: h[i + 1] after token i, e before token 0, and the decay over all
                pair_t w[K][2], h[K + 1][2], up[2], down[2], e[2];
                {
                    pair_t step[K];
                    load_pairs<K>(sD + here, step);
#pragma unroll
                    for (int i = 0; i < K; ++i)
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            w[i][p] = decay2_fine(step[i], rate[p]);
                            const pair_t b = mul2(u[i], B[i][p]);
                            h[i + 1][p] = i == 0 ? b : mad2(w[i][p], h[i][p], b);
                            up[p] = i == 0 ? w[i][p] : mul2(up[p], w[i][p]);
                        }
                }
#pragma unroll
                for (int i = K - 1; i >= 0; --i)
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        e[p] = mul2(w[i][p], i == K - 1 ? mul2(C[i][p], gg[i]) : mad2(C[i][p], gg[i], e[p]));
                // scans over the token groups.  The first group takes in the state kept for the chunk, the last the
                // gradient that follows it; their decay then counts as zero, so that a group that has seen
                // everything before it adds nothing more (a shuffle from beyond the edge returns the lane's own value).
                const bool scans = within_range<TL>(up);
                pair_t in[2];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    in[p] = h[K][p];
                    down[p] = up[p];
                    in[p] = mad2(up[p], tl == 0 ? entry[p] : 0, in[p]);
                    e[p] = mad2(down[p], tl == TL - 1 ? leave[p] : 0, e[p]);
                    up[p] = tl == 0 ? 0 : up[p];
                    down[p] = tl == TL - 1 ? 0 : down[p];
                }
#pragma unroll
                for (int off = 1; off < TL; off *= 2)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        in[p] = mad2(up[p], shift_up(in[p], off * LN), in[p]);
                        e[p] = mad2(down[p], shift_down(e[p], off * LN), e[p]);
                        if (2 * off < TL) {
                            up[p] = mul2(up[p], shift_up(up[p], off * LN));
                            down[p] = mul2(down[p], shift_down(down[p], off * LN));
                        }
                    }
                if (!scans) {
                    // growing rates: group after group, token after token, no product of decays
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        pair_t now = entry[p];
#pragma unroll 1
                        for (int t = 0; t < TL; ++t) {
#pragma unroll
                            for (int i = 0; i < K; ++i) now = mad2(w[i][p], now, mul2(u[i], B[i][p]));
                            if (tl == t) in[p] = now;
                            now = from_lane(now, t * LN + sub);
                        }
                        now = leave[p];
#pragma unroll 1
                        for (int t = TL - 1; t >= 0; --t) {
#pragma unroll
                            for (int i = K - 1; i >= 0; --i) now = mul2(w[i][p], mad2(C[i][p], gg[i], now));
                            if (tl == t) e[p] = now;
                            now = from_lane(now, t * LN + sub);
                        }
                    }
                }
                __syncwarp();
                if (tl == 0) {
                    *reinterpret_cast<pair_t*>(kept) = e[0];
                    *reinterpret_cast<pair_t*>(kept + 2) = e[1];
                }
                // the true states
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    in[p] = shift_up(in[p], LN);
                    e[p] = shift_down(e[p], LN);
                    in[p] = tl == 0 ? entry[p] : in[p];
                    e[p] = tl == TL - 1 ? leave[p] : e[p];
                    h[0][p] = in[p];
#pragma unroll
                    for (int i = 0; i < K; ++i) {
                        in[p] = mul2(in[p], w[i][p]);
                        h[i + 1][p] = add2(h[i + 1][p], in[p]);
                    }
                }
                if (GATE)
#pragma unroll
                    for (int i = 0; i < K; ++i) y[i] = halves(mad2(C[i][1], h[i + 1][1], mul2(C[i][0], h[i + 1][0])));
                // backwards from the true gradient
                pair_t* sums = reinterpret_cast<pair_t*>(smem + G.dA + ((c * G.slices + q) * 32 + lane) * 4);
                pair_t dA[2] = {sums[0], sums[1]}, step[K];
                load_pairs<K>(sD + here, step);
#pragma unroll
                for (int i = K - 1; i >= 0; --i) {
                    pair_t to_u, to_d;
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const pair_t now = mad2(C[i][p], gg[i], e[p]);
                        e[p] = mul2(w[i][p], now);
                        dB[i][p] = mad2(now, u[i], dB[i][p]);
                        dC[i][p] = mad2(h[i + 1][p], gg[i], dC[i][p]);
                        to_u = p == 0 ? mul2(now, B[i][p]) : mad2(now, B[i][p], to_u);
                        const pair_t moved = mul2(e[p], h[i][p]);
                        to_d = p == 0 ? mul2(moved, rate[p]) : mad2(moved, rate[p], to_d);
                        dA[p] = mad2(moved, step[i], dA[p]);
                    }
                    du[i] = halves(to_u);
                    dd[i] = halves(to_d);
                }
                sums[0] = dA[0];
                sums[1] = dA[1];
                // this lane's token
                float ty = GATE ? sum_to_lane<K>(y, sub) : 0.0f, tu = sum_to_lane<K>(du, sub), td = sum_to_lane<K>(dd, sub);
                const int at = place(c, lane);
                if (G.slices > 1) {
                    if (q > 0) { ty += smem[G.y + at]; tu += smem[G.du + at]; td += smem[G.dd + at]; }
                    smem[G.y + at] = ty; smem[G.du + at] = tu; smem[G.dd + at] = td;
                }
                if (q == G.slices - 1) {
                    __syncwarp();     // the chunk's inputs of this channel give way to its gradients
#if PD_MODE == 2
                    td *= 0.6931471805599453f;     // rates are in units of log2(e)
#endif
                    const float tx = sX[at], tstep = sD[at].x, tg = sG[at].x, skip = smem[G.skip + c];
                    sX[at] = tu * tstep + skip * tg;
                    sS[at] *= td + tu * tx;
                    if (GATE) sZ[at] *= ty + skip * tx;
                }
            }
            // dB and dC over the block's warps, in order
            float* red = smem + G.red;
            constexpr int kStep = 2 * kWide + 4;
#pragma unroll
            for (int i = 0; i < K; ++i) {
                float* to = red + (warp * kRow + tl * K + i) * kStep + sub * 4;
                *reinterpret_cast<ulonglong2*>(to) = make_ulonglong2(dB[i][0], dB[i][1]);
                *reinterpret_cast<ulonglong2*>(to + kWide) = make_ulonglong2(dC[i][0], dC[i][1]);
            }
            __syncthreads();
#pragma unroll
            for (int v = tid; v < kRow * 2 * LN; v += kGradThreads) {
                const int t = v / (2 * LN), part = v % (2 * LN) * 4;
                float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int k2 = 0; k2 < PD_SCAN_GRAD_WARPS; ++k2) {
                    const float4 p = *reinterpret_cast<const float4*>(red + (k2 * kRow + t) * kStep + part);
                    total.x += p.x; total.y += p.y; total.z += p.z; total.w += p.w;
                }
                if (from + t < end) {
                    const int which = part / kWide;
                    *reinterpret_cast<float4*>(bc_out + ((from + t) * 2 + which) * G.pad + q * kWide + part % kWide) = total;
                }
            }
            if (q + 1 < G.slices) __syncthreads();
        }
        for (int t = st; t < kRow; t += rows) {
            const int n = from + t < end ? left : 0;
            const int64_t at = (from + t) * a.channels + c0 + c4;
            const int row = place(c4, t);
            float vx[4], vd[4], vz[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = row + i * kRow;
                vx[i] = sX[p];
                vd[i] = sS[p];
                if (GATE) vz[i] = sZ[p];
                if (i < n) dbias[i] += vd[i];
            }
            put4((T*)a.dx + at, a.vec, n, vx);
            put4((T*)a.ddelta + at, a.vec, n, vd);
            if (GATE) put4((T*)a.dz + at, a.vec, n, vz);
        }
        __syncthreads();
    }
    __syncthreads();
    if (a.dinitial)
        for (int i = tid; i < count * G.pad; i += kGradThreads)
            if (i % G.pad < a.state) a.dinitial[(s * a.channels + c0 + i / G.pad) * a.state + i % G.pad] = smem[G.carry + i];
    // the sequence's sums: dA over the token groups, dbias and dskip over the staging threads of a channel
    float* out = a.partial_params + (s * a.channels + c0) * (a.state + 2);
    for (int i = tid; i < count * a.state; i += kGradThreads) {
        const int c = i / a.state, n = i % a.state;
        const float* p = smem + G.dA + (c * G.slices + n / kWide) * 128 + n % kWide / 4 * 4 + n % 4;
        float total = 0.0f;
#pragma unroll
        for (int j = 0; j < TL; ++j) total += p[j * LN * 4];
        out[c * (a.state + 2) + n] = total;
    }
    float* part = smem + G.red;      // (staging row, channel, 2)
    if (stages)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            part[(st * G.channels + c4 + i) * 2] = dbias[i];
            part[(st * G.channels + c4 + i) * 2 + 1] = dskip[i];
        }
    __syncthreads();
    for (int i = tid; i < count * 2; i += kGradThreads) {
        float total = 0.0f;
        for (int t = 0; t < rows; ++t) total += part[t * G.channels * 2 + i];
        out[i / 2 * (a.state + 2) + a.state + i % 2] = total;
    }
}

// dB and dC: the tiles of a group added up in order, four states per thread
template <class T>
__global__ void __launch_bounds__(256) pd_selective_scan_sum_bc_kernel(PdScanArgs a, int pad, int tiles) {
    const int64_t wide = a.tok.rows * 2 * pad;
    const int64_t at = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 4, g = blockIdx.y;
    if (at >= wide) return;
    const int64_t r = at / (2 * pad);
    const int n = (int)(at - r * 2 * pad), which = n >= pad, first = n - which * pad;
    const float* p = a.partial_bc + g * tiles * wide + at;
    float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (a.tok.offsets) {        // no tile has sums of a row of no sequence
        int64_t head, tail;
        free_rows(a.tok, head, tail);
        if (r < head || r >= tail) tiles = 0;
    }
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
        const float4 q = *reinterpret_cast<const float4*>(p + t * wide);
        total.x += q.x; total.y += q.y; total.z += q.z; total.w += q.w;
    }
    const float v[4] = {total.x, total.y, total.z, total.w};
    T* to = (T*)(which ? a.dC : a.dB) + (r * a.groups + g) * a.state;
#pragma unroll
    for (int i = 0; i < 4; ++i) if (first + i < a.state) store1(to + first + i, v[i]);
}

// dA, dbias and dskip: the sequences added up in order; the blocks behind clear the rows of no sequence
template <class T>
__global__ void __launch_bounds__(128) pd_selective_scan_sum_params_kernel(PdScanArgs a) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t wide = a.channels * (a.state + 2);
    const int64_t part = blockIdx.x - (int64_t)(gridDim.x - a.free_blocks);
    if (part >= 0) {
        clear_free_rows(a.tok, a.channels, (T*)a.dx, part, a.free_blocks);
        clear_free_rows(a.tok, a.channels, (T*)a.ddelta, part, a.free_blocks);
        if (a.dz) clear_free_rows(a.tok, a.channels, (T*)a.dz, part, a.free_blocks);
        return;
    }
    if (i >= wide) return;
    float total = 0.0f;
#pragma unroll 4
    for (int64_t s = 0; s < a.tok.seqs; ++s) total += a.partial_params[s * wide + i];
    const int64_t c = i / (a.state + 2);
    const int k = (int)(i % (a.state + 2));
    if (k < a.state) a.dA[c * a.state + k] = total;
    else if (k == a.state) { if (a.dbias) a.dbias[c] = total; }
    else if (a.dskip) a.dskip[c] = total;
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
int64_t blocks_for(int64_t threads, int block) { return (threads + block - 1) / block; }

// Up to 48 KB of shared memory need no leave; beyond, a kernel is given all that a block may have, always the same: calls
// of other sizes on other threads share its limit, and one that lowered it would have the next launch refused.
template <class K>
cudaError_t allow_smem(K kernel, int bytes) {
    return bytes <= 48 * 1024 ? cudaSuccess
                              : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
}

template <class K>
cudaError_t describe(K kernel, int threads, int bytes, PdScanReport* to) {
    cudaFuncAttributes attr;
    cudaError_t err = allow_smem(kernel, bytes);
    if (err == cudaSuccess) err = cudaFuncGetAttributes(&attr, kernel);
    int blocks = 0;
    if (err == cudaSuccess) err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, threads, bytes);
    if (err != cudaSuccess) {
        cudaGetLastError();
        return err;
    }
    to->registers = attr.numRegs;
    to->static_smem = (int)attr.sharedSizeBytes;
    to->blocks_per_sm = blocks;
    return cudaSuccess;
}

template <class F>
cudaError_t by_type(int type, F f) {
    if (type == PD_TYPE_F32) return f(float());
    if (type == PD_TYPE_F16) return f(__half());
    return f(__nv_bfloat16());
}
template <int V> struct Int { static constexpr int value = V; };
template <class F>
cudaError_t by_width(int width, F f) {
    return width == 2 ? f(Int<2>()) : width == 3 ? f(Int<3>()) : f(Int<4>());
}
template <class F>
cudaError_t by_lanes(int state, F f) {
    switch (pd_scan_lanes(state)) {
        case 1: return f(Int<1>());
        case 2: return f(Int<2>());
        case 4: return f(Int<4>());
        case 8: return f(Int<8>());
        default: return f(Int<16>());
    }
}
// f(element, width, vector) for the call's type, width and alignment
template <class F>
cudaError_t by_conv(const PdConvArgs& a, F f) {
    return by_type(a.type, [&](auto e) {
        return by_width(a.width, [&](auto w) {
            return a.vec > 1 ? f(e, w, Int<4>()) : f(e, w, Int<1>());
        });
    });
}

cudaError_t launch_conv(const PdConvArgs& a, cudaStream_t st) {
    return by_conv(a, [&](auto e, auto w, auto v) {
        using T = decltype(e);
        const int64_t lanes = (a.channels + v.value - 1) / v.value;
        const int64_t jobs = (a.tok.rows + a.run - 1) / a.run + (a.final_state ? a.tok.seqs : 0);
        constexpr int W = decltype(w)::value, V = decltype(v)::value;
        auto kernel = a.silu ? pd_causal_conv_kernel<T, W, V, true> : pd_causal_conv_kernel<T, W, V, false>;
        if (a.report) return describe(kernel, 256, 0, a.report);
        if (lanes * jobs == 0) return cudaSuccess;
        kernel<<<(unsigned)blocks_for(lanes * jobs, 256), 256, 0, st>>>(a);
        return cudaGetLastError();
    });
}
cudaError_t launch_conv_step(const PdConvArgs& a, cudaStream_t st) {
    return by_conv(a, [&](auto e, auto w, auto v) {
        using T = decltype(e);
        const int64_t lanes = (a.channels + v.value - 1) / v.value;
        auto kernel = pd_causal_conv_step_kernel<T, decltype(w)::value, decltype(v)::value>;
        if (a.report) return describe(kernel, 128, 0, a.report);
        if (a.tok.seqs == 0) return cudaSuccess;
        const dim3 grid((unsigned)blocks_for(lanes, 128), (unsigned)(a.tok.seqs < 65535 ? a.tok.seqs : 65535));
        kernel<<<grid, 128, 0, st>>>(a);
        return cudaGetLastError();
    });
}
cudaError_t launch_conv_grad(const PdConvArgs& a, cudaStream_t st) {
    return by_conv(a, [&](auto e, auto w, auto v) {
        using T = decltype(e);
        constexpr int W = decltype(w)::value, V = decltype(v)::value;
        const int64_t lanes = (a.channels + V - 1) / V;
        const dim3 block(32, 8), grid((unsigned)blocks_for(lanes, 32), (unsigned)a.row_blocks);
        auto kernel = a.silu ? pd_causal_conv_grad_kernel<T, W, V, true> : pd_causal_conv_grad_kernel<T, W, V, false>;
        if (a.report) return describe(kernel, 256, 256 * V * sizeof(float), a.report);
        kernel<<<grid, block, 256 * V * sizeof(float), st>>>(a);
        cudaError_t err = cudaGetLastError();
        if (err != cudaSuccess) return err;
        pd_causal_conv_sum_kernel<W><<<(unsigned)blocks_for(a.channels * (W + 1), 128), 128, 0, st>>>(a);
        return cudaGetLastError();
    });
}

cudaError_t launch_scan(const PdScanArgs& a, cudaStream_t st) {
    return by_type(a.type, [&](auto e) {
        using T = decltype(e);
        return by_lanes(a.state, [&](auto ln) -> cudaError_t {
            constexpr int LN = decltype(ln)::value;
            const bool full = a.state == 4 * LN;
            auto run = [&](auto nch) -> cudaError_t {
                constexpr int NCH = decltype(nch)::value;
                constexpr PdScanShape G(LN, NCH, sizeof(T));
                const int64_t per = a.channels / a.groups, tiles = (per + G.channels - 1) / G.channels * a.groups;
                auto kernel = full ? pd_selective_scan_kernel<T, LN, NCH, true, false> : pd_selective_scan_kernel<T, LN, NCH, false, false>;
                if (a.report) return describe(kernel, kScanThreads, G.bytes, a.report);
                if (a.ends && a.segments > 0) {
                    auto first = full ? pd_selective_scan_kernel<T, LN, NCH, true, true> : pd_selective_scan_kernel<T, LN, NCH, false, true>;
                    cudaError_t err = allow_smem(first, G.bytes);
                    if (err != cudaSuccess) return err;
                    first<<<(unsigned)(tiles * a.segments), kScanThreads, G.bytes, st>>>(a);
                    err = cudaGetLastError();
                    if (err != cudaSuccess) return err;
                }
                const int64_t blocks = tiles * (a.segments + a.free_blocks);
                if (blocks == 0) return cudaSuccess;
                cudaError_t err = allow_smem(kernel, G.bytes);
                if (err != cudaSuccess) return err;
                kernel<<<(unsigned)blocks, kScanThreads, G.bytes, st>>>(a);
                return cudaGetLastError();
            };
            if constexpr (LN == 16) {
                return run(Int<2>());      // (one channel per lane would leave a warp two)
            } else {
                if constexpr (LN >= 4) {
                    if (a.per_warp == 2) return run(Int<2>());
                }
                return run(Int<1>());
            }
        });
    });
}
cudaError_t launch_scan_step(const PdScanArgs& a, cudaStream_t st) {
    return by_type(a.type, [&](auto e) {
        using T = decltype(e);
        return by_lanes(a.state, [&](auto ln) {
            constexpr int LN = decltype(ln)::value;
            const bool vec = a.state == 4 * LN && a.vec_states && a.vec_params;
            auto kernel = vec ? pd_selective_scan_step_kernel<T, LN, true> : pd_selective_scan_step_kernel<T, LN, false>;
            const int threads = 32 * pd_step_warps(a.channels, a.groups, a.state, a.tok.seqs);
            if (a.report) return describe(kernel, threads, 0, a.report);
            if (a.tok.seqs == 0) return cudaSuccess;
            const dim3 grid((unsigned)pd_step_blocks(a.channels, a.groups, a.state, a.tok.seqs),
                            (unsigned)((a.tok.seqs + a.run - 1) / a.run));
            kernel<<<grid, threads, 0, st>>>(a);
            return cudaGetLastError();
        });
    });
}
cudaError_t launch_scan_grad(const PdScanArgs& a, cudaStream_t st) {
    return by_type(a.type, [&](auto e) {
        using T = decltype(e);
        auto run = [&](auto ln) -> cudaError_t {
            constexpr int LN = decltype(ln)::value;
            const bool one = a.state <= 4 * LN;
            const PdGradShape<LN, false> G(a.state, a.per_warp, sizeof(T));
            const int64_t per = a.channels / a.groups, tiles = (per + G.channels - 1) / G.channels;
            const int64_t blocks = tiles * a.groups * a.tok.seqs;
            if (blocks > 0 || a.report) {
                auto kernel = a.z ? pd_selective_scan_grad_kernel<T, LN, true, true> : pd_selective_scan_grad_kernel<T, LN, false, true>;
                if constexpr (LN == 4)
                    if (!one) kernel = a.z ? pd_selective_scan_grad_kernel<T, LN, true, false> : pd_selective_scan_grad_kernel<T, LN, false, false>;
                if (a.report) return describe(kernel, kGradThreads, G.bytes, a.report);
                cudaError_t err = allow_smem(kernel, G.bytes);
                if (err != cudaSuccess) return err;
                kernel<<<(unsigned)blocks, kGradThreads, G.bytes, st>>>(a);
                err = cudaGetLastError();
                if (err != cudaSuccess) return err;
            }
            const int64_t fours = a.tok.rows * 2 * G.pad / 4;
            if (fours > 0) {
                const dim3 grid((unsigned)blocks_for(fours, 256), (unsigned)a.groups);
                pd_selective_scan_sum_bc_kernel<T><<<grid, 256, 0, st>>>(a, G.pad, (int)tiles);
                cudaError_t err = cudaGetLastError();
                if (err != cudaSuccess) return err;
            }
            pd_selective_scan_sum_params_kernel<T><<<(unsigned)(blocks_for(a.channels * (a.state + 2), 128) + a.free_blocks), 128, 0, st>>>(a);
            return cudaGetLastError();
        };
        return a.state <= 4 ? run(Int<1>()) : a.state <= 8 ? run(Int<2>()) : run(Int<4>());
    });
}

}  // namespace

const PdScanTable* PD_SCAN_TABLE() {
    static const PdScanTable table = {launch_conv, launch_conv_step, launch_conv_grad, launch_scan, launch_scan_step, launch_scan_grad};
    return &table;
}
