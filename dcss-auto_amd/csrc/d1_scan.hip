// d1ops: a gated linear recurrence over long sequences, its backward pass, gfx950.
//
// With z = sigmoid(gate), a = 1 - z, and m = 0 where a reset drops what was before (1 elsewhere):
//   h[t] = a[t] m[t] h[t-1] + z[t] x[t]
// backward, from the end, with C[t] = a[t] m[t] G[t] what a step hands to the one before it:
//   G[t] = dh[t] + C[t+1];  dx = z G;  dgate = G (x - m h[t-1]) z a;  dstate = C[0]
//
// A step's map h -> a h + b composes: (A, B) then (A', B') is (A A', A' B + B'). A wave takes STEPS rows of 64 VEC channels
// into registers, one channel set a lane, and forms their composite; the waves of a workgroup, whose rows follow each
// other, exchange composites through LDS and each then walks its rows once more from the state before them. A
// workgroup goes on along its sequence, so every input is read once; up to 8 steps are a single wave's. Where channels
// alone would leave CUs idle, the sequence is cut into segments: a first launch forms the segments' composites and the
// second starts each segment from those before it (no workgroup waits for another). The backward pass reads no h: forward
// keeps the fp32 state before every MARK-th step and the backward pass makes the states between again, which costs 4 bytes
// a channel in MARK steps and gives dgate from states that were never rounded to 16 bits.
// A product A is -1 (sign bit) once a reset lies in it: what comes before is dropped, even where it is not finite.
// Everything is computed in fp32. Bound by memory, in 16 bits nearly as much by the instructions (some 35 an element
// forward, two thirds of them the sigmoid's): 128 steps of 8,192 x 256 bf16 take 378 us forward (1.6 GB, 4.3 TB/s) and 652
// backward (2.7 GB, 4.1 TB/s; a large copy 4.8), 65,537 steps of 1,024 channels, cut, 78 + 100 us forward, 77 + 170 backward.
#include <type_traits>

#include "d1_rows.h"

namespace d1o {

constexpr int MARK = 64;
constexpr int SCAN_STEPS = 8, SCAN_WAVES = MARK / SCAN_STEPS;

struct Scan {
    const void *x, *gate, *dh;
    void *h, *dx, *dgate;
    const uint8_t *reset;
    const float *state, *dlast;
    float *last, *dstate, *marks;
    float *parts;                         // composites of the segments: A then B, [segments][rows * width] each
    int64_t x_t, x_n, gate_t, gate_n, dh_t, dh_n, h_t, h_n, dx_t, dx_n, dgate_t, dgate_n, reset_t, reset_n;
    int64_t steps, cells;                 // cells = rows * width
    uint32_t units;                       // the launch's rows * columns
    int32_t width, columns;               // columns: workgroups (waves, where each is on its own) beside each other on one row's channels
    int32_t past;                         // results past the caches
    int32_t segments, seg;                // seg: steps of a segment, a multiple of MARK
};

template <int VEC>
struct Cells {
    int64_t row;
    int32_t at;                           // first channel of the lane
    bool any;
};
// the lane's channels; those past the end are moved back over it (both lanes then store the same values)
template <int VEC>
__device__ __forceinline__ Cells<VEC> cells_of(const Scan &s, uint32_t unit) {
    Cells<VEC> c;
    c.row = unit / s.columns;
    const int at = ((int)(unit % s.columns) * 64 + (threadIdx.x & 63)) * VEC;
    c.any = at < s.width;
    c.at = at < s.width - VEC ? at : s.width - VEC;
    return c;
}

// z = sigmoid(g) and a = sigmoid(-g), each exact to a few ulp where it is small too: 1 / (1 + e) and e / (1 + e) with
// e = e^-|g|, which is 2^p of the rounded product p = -|g| log2 e times what the rounding dropped. A bf16 gate's product with
// 16 bits of log2 e is exact, which leaves the constant's own rest. (A NaN passes through p. The bounds on the rest are for
// gates whose product passes fp32's range, where e is 0: it is NaN for -inf, infinite below -2.36e38.) The reciprocal is
// refined: one that is off to one side adds up over thousands of steps.
template <class T>
__device__ __forceinline__ void gate_of(float g, float &z, float &a) {
    const float y = -fabsf(g);
    float p, rest;
    if constexpr (__is_same(T, __bf16)) {
        p = y * 1.44268798828125f;
        rest = y * (7.0526077e-06f * 0.693147181f);
    } else {
        p = y * 1.44269504f;
        rest = __builtin_fmaf(y, 1.92596299e-8f, __builtin_fmaf(y, 1.44269504f, -p)) * 0.693147181f;
    }
    float e = __builtin_amdgcn_exp2f(p);
    e = __builtin_fmaf(e, fminf(fmaxf(rest, -1.f), 1.f), e);
    float big = __builtin_amdgcn_rcpf(1.f + e);
    big = __builtin_fmaf(__builtin_fmaf(-(1.f + e), big, 1.f), big, big);
    const float small = e * big;
    z = g >= 0.f ? big : small;
    a = g >= 0.f ? small : big;
}

// the bits of the steps that drop what was before: step first + j in bit j
template <int STEPS>
__device__ __forceinline__ uint32_t resets_of(const Scan &s, int64_t row, int64_t first, int64_t end) {
    if (!s.reset) return 0;
    const int j = threadIdx.x & 63;
    const bool r = j < STEPS && first + j < end && s.reset[(first + j) * s.reset_t + row * s.reset_n];
    return (uint32_t)__ballot(r);
}

// the state after the composite (a, b)
__device__ __forceinline__ float after(float a, float b, float h) { return __float_as_int(a) < 0 ? b : __builtin_fmaf(a, h, b); }

// A row's address is the wave's, a lane's place in it 32 bits of bytes.
template <class T>
__device__ __forceinline__ T *lane_of(T *row, uint32_t at) { return (T *)((char *)row + at * (uint32_t)sizeof(T)); }
template <int STEPS, class T, int VEC>
__device__ __forceinline__ void rows_of(const T *p, int64_t st, uint32_t at, int64_t first, int64_t end, Pack<T, VEC> *out) {
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        const int64_t t = first + j < end ? first + j : end - 1;
        out[j] = load<T, VEC>(lane_of((const T *)(p + t * st), at));
    }
}
template <class T, int VEC>
__device__ __forceinline__ void put_row(T *p, const Pack<T, VEC> &a, int past) {
    if constexpr (sizeof(a) >= 4) {
        if (past) return store_past<T, VEC>(p, a);
    }
    store<T, VEC>(p, a);
}
// the composite of the segments `order(k)` for k in [lo, hi), which follow each other
template <int VEC, class Order>
__device__ __forceinline__ void join(const Scan &s, int64_t row0, uint32_t at, int lo, int hi, Order order, float *a, float *b) {
#pragma unroll
    for (int v = 0; v < VEC; v++) a[v] = 1.f, b[v] = 0.f;
    constexpr int AT_ONCE = 8;
    for (int k = lo; k < hi; k += AT_ONCE) {
        Pack<float, VEC> pa[AT_ONCE], pb[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int from = order(k + u < hi ? k + u : hi - 1);
            pa[u] = load<float, VEC>(lane_of(s.parts + from * s.cells + row0, at));
            pb[u] = load<float, VEC>(lane_of(s.parts + (s.segments + from) * s.cells + row0, at));
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
            if (k + u < hi)
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    b[v] = after(pa[u].v[v], pb[u].v[v], b[v]);
                    a[v] = __float_as_int(pa[u].v[v]) < 0 ? -1.f : a[v] * pa[u].v[v];
                }
    }
}

// ---- a wave alone: up to STEPS steps

template <class T, int VEC, int STEPS>
__global__ __launch_bounds__(256) void k_scan_own_fwd(const Scan s) {
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= s.units) return;
    const Cells<VEC> c = cells_of<VEC>(s, unit);
    const int64_t row0 = c.row * s.width;
    Pack<float, VEC> h;
#pragma unroll
    for (int v = 0; v < VEC; v++) h.v[v] = 0.f;
    if (s.state) h = load<float, VEC>(lane_of(s.state + row0, c.at));
    Pack<T, VEC> px[STEPS], pg[STEPS];
    rows_of<STEPS, T, VEC>((const T *)s.gate + c.row * s.gate_n, s.gate_t, c.at, 0, s.steps, pg);
    rows_of<STEPS, T, VEC>((const T *)s.x + c.row * s.x_n, s.x_t, c.at, 0, s.steps, px);
    const uint32_t drop = resets_of<STEPS>(s, c.row, 0, s.steps);
    if (!c.any) return;
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        if (j >= s.steps) break;
        Pack<T, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z, a;
            gate_of<T>((float)pg[j].v[v], z, a);
            h.v[v] = __builtin_fmaf(a, drop >> j & 1 ? 0.f : h.v[v], z * (float)px[j].v[v]);
            o.v[v] = (T)h.v[v];
        }
        put_row<T, VEC>(lane_of((T *)s.h + c.row * s.h_n + j * s.h_t, c.at), o, s.past);
    }
    if (s.last) store<float, VEC>(lane_of(s.last + row0, c.at), h);
}

template <class T, int VEC, int STEPS>
__global__ __launch_bounds__(256) void k_scan_own_bwd(const Scan s) {
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= s.units) return;
    const Cells<VEC> c = cells_of<VEC>(s, unit);
    const int64_t row0 = c.row * s.width;
    Pack<float, VEC> C, h;
#pragma unroll
    for (int v = 0; v < VEC; v++) C.v[v] = h.v[v] = 0.f;
    if (s.dlast) C = load<float, VEC>(lane_of(s.dlast + row0, c.at));
    if (s.state) h = load<float, VEC>(lane_of(s.state + row0, c.at));
    Pack<T, VEC> px[STEPS], pg[STEPS], pd[STEPS];
    rows_of<STEPS, T, VEC>((const T *)s.gate + c.row * s.gate_n, s.gate_t, c.at, 0, s.steps, pg);
    rows_of<STEPS, T, VEC>((const T *)s.x + c.row * s.x_n, s.x_t, c.at, 0, s.steps, px);
    rows_of<STEPS, T, VEC>((const T *)s.dh + c.row * s.dh_n, s.dh_t, c.at, 0, s.steps, pd);
    const uint32_t drop = resets_of<STEPS>(s, c.row, 0, s.steps);
    if (!c.any) return;
    float a[STEPS][VEC], z[STEPS][VEC], e[STEPS][VEC];
#pragma unroll
    for (int j = 0; j < STEPS; j++)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const float in = (float)px[j].v[v], before = drop >> j & 1 ? 0.f : h.v[v];
            gate_of<T>((float)pg[j].v[v], z[j][v], a[j][v]);
            e[j][v] = (in - before) * (z[j][v] * a[j][v]);
            h.v[v] = __builtin_fmaf(a[j][v], before, z[j][v] * in);
        }
#pragma unroll
    for (int j = STEPS - 1; j >= 0; j--) {
        if (j >= s.steps) continue;
        Pack<T, VEC> ox, og;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const float g = (float)pd[j].v[v] + C.v[v];
            ox.v[v] = (T)(z[j][v] * g);
            og.v[v] = (T)(g * e[j][v]);
            C.v[v] = drop >> j & 1 ? 0.f : a[j][v] * g;
        }
        put_row<T, VEC>(lane_of((T *)s.dx + c.row * s.dx_n + j * s.dx_t, c.at), ox, s.past);
        put_row<T, VEC>(lane_of((T *)s.dgate + c.row * s.dgate_n + j * s.dgate_t, c.at), og, s.past);
    }
    if (s.dstate) store<float, VEC>(lane_of(s.dstate + row0, c.at), C);
}

// ---- the waves of a workgroup on one sequence

// Workgroups go round the eight chiplets; neighbours on one row share cache lines where its width is odd, so a chiplet
// takes units in a row.
__device__ __forceinline__ uint32_t unit_of(const Scan &s) {
    const uint32_t b = blockIdx.x, whole = s.units & ~7u, each = whole >> 3;
    return b < whole ? (b & 7u) * each + (b >> 3) : b;
}
template <int VEC>
struct Exchange {
    float v[SCAN_WAVES][VEC][64];
};
// The waves' reset flags, as bits, from what each has put into LDS before the last barrier
__device__ __forceinline__ uint32_t flags_of(const uint32_t *flags, int waves) {
    return (uint32_t)__ballot((int)(threadIdx.x & 63) < waves && flags[threadIdx.x & (SCAN_WAVES - 1)]);
}
// `state` past wave w's composite; `some`: whether any wave has a reset
__device__ __forceinline__ float past_wave(float a, float b, float state, bool some) {
    return some ? after(a, b, state) : __builtin_fmaf(a, state, b);
}

// Forward. PART: the composites of all segments but the last alone.
template <class T, int VEC, bool PART>
__global__ __launch_bounds__(64 * SCAN_WAVES) void k_scan_fwd(const Scan s) {
    constexpr int STEPS = SCAN_STEPS;
    __shared__ Exchange<VEC> ex[2][2];
    __shared__ uint32_t flags[2][SCAN_WAVES];
    const Cells<VEC> c = cells_of<VEC>(s, unit_of(s));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    const int64_t begin = (int64_t)blockIdx.y * s.seg, end = begin + s.seg < s.steps ? begin + s.seg : s.steps;
    const T *x = (const T *)s.x + c.row * s.x_n, *gate = (const T *)s.gate + c.row * s.gate_n;
    T *out = (T *)s.h + c.row * s.h_n;
    const int64_t row0 = c.row * s.width;
    float A[VEC], h[VEC];                 // the workgroup's composite so far (PART), or the state
    int turn = 0;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        A[v] = 1.f;
        h[v] = PART ? 0.f : s.state ? s.state[row0 + c.at + v] : 0.f;
    }
    if (!PART && blockIdx.y) {            // the state that the segments before leave: each wave joins a share of them
        const int n = blockIdx.y, per = (n + waves - 1) / waves, lo = wave * per < n ? wave * per : n, hi = lo + per < n ? lo + per : n;
        float a[VEC], b[VEC];
        join<VEC>(s, row0, c.at, lo, hi, [](int k) { return k; }, a, b);
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[0][0].v[wave][v][lane] = a[v];
            ex[0][1].v[wave][v][lane] = b[v];
        }
        __syncthreads();
        for (int w = 0; w < waves; w++)
#pragma unroll
            for (int v = 0; v < VEC; v++) h[v] = after(ex[0][0].v[w][v][lane], ex[0][1].v[w][v][lane], h[v]);
        turn = 1;
    }
    for (int64_t tile = begin; tile < end; tile += waves * STEPS, turn ^= 1) {
        const int64_t first = tile + wave * STEPS;
        float a[STEPS][VEC], b[STEPS][VEC], ca[VEC], cb[VEC];
        uint32_t drop = 0;
#pragma unroll
        for (int v = 0; v < VEC; v++) ca[v] = 1.f, cb[v] = 0.f;
        const bool plain = first + STEPS <= end;
        if (first < end) {
            Pack<T, VEC> px[STEPS], pg[STEPS];
            rows_of<STEPS, T, VEC>(gate, s.gate_t, c.at, first, end, pg);
            rows_of<STEPS, T, VEC>(x, s.x_t, c.at, first, end, px);
            drop = resets_of<STEPS>(s, c.row, first, end);
#pragma unroll
            for (int j = 0; j < STEPS; j++)
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    float z;
                    gate_of<T>((float)pg[j].v[v], z, a[j][v]);
                    b[j][v] = z * (float)px[j].v[v];
                }
            if (plain && !drop) {
#pragma unroll
                for (int j = 0; j < STEPS; j++)
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        ca[v] *= a[j][v];
                        cb[v] = __builtin_fmaf(a[j][v], cb[v], b[j][v]);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < STEPS; j++)
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        const bool on = first + j < end, cut = drop >> j & 1;
                        a[j][v] = on ? a[j][v] : 1.f;
                        b[j][v] = on ? b[j][v] : 0.f;
                        cb[v] = __builtin_fmaf(a[j][v], cut ? 0.f : cb[v], b[j][v]);
                        ca[v] = cut ? -1.f : ca[v] * a[j][v];
                    }
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[turn][0].v[wave][v][lane] = ca[v];
            ex[turn][1].v[wave][v][lane] = cb[v];
        }
        if (lane == 0) flags[turn][wave] = drop;
        __syncthreads();
        const bool some = flags_of(flags[turn], waves) != 0;
        if (!PART && s.marks && tile && wave == 0 && c.any) {
            Pack<float, VEC> m;
#pragma unroll
            for (int v = 0; v < VEC; v++) m.v[v] = h[v];
            store<float, VEC>(lane_of(s.marks + (tile / MARK - 1) * s.cells + row0, c.at), m);
        }
        float mine[VEC];
        for (int w = 0; w < waves; w++) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                if (w == wave) mine[v] = h[v];
                const float pa = ex[turn][0].v[w][v][lane], pb = ex[turn][1].v[w][v][lane];
                h[v] = past_wave(pa, pb, h[v], some);
                if (PART) A[v] = __float_as_int(pa) < 0 ? -1.f : A[v] * pa;
            }
        }
        if (!PART && first < end && c.any) {
            if (plain && !drop) {
#pragma unroll
                for (int j = 0; j < STEPS; j++) {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        mine[v] = __builtin_fmaf(a[j][v], mine[v], b[j][v]);
                        o.v[v] = (T)mine[v];
                    }
                    put_row<T, VEC>(lane_of(out + (first + j) * s.h_t, c.at), o, s.past);
                }
            } else {
#pragma unroll
                for (int j = 0; j < STEPS; j++) {
                    if (first + j >= end) break;
                    Pack<T, VEC> o;
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        mine[v] = __builtin_fmaf(a[j][v], drop >> j & 1 ? 0.f : mine[v], b[j][v]);
                        o.v[v] = (T)mine[v];
                    }
                    put_row<T, VEC>(lane_of(out + (first + j) * s.h_t, c.at), o, s.past);
                }
            }
        }
    }
    if (wave || !c.any) return;
    if (PART) {
        Pack<float, VEC> pa, pb;
#pragma unroll
        for (int v = 0; v < VEC; v++) pa.v[v] = A[v], pb.v[v] = h[v];
        store<float, VEC>(lane_of(s.parts + blockIdx.y * s.cells + row0, c.at), pa);
        store<float, VEC>(lane_of(s.parts + (s.segments + blockIdx.y) * s.cells + row0, c.at), pb);
    } else if (s.last && end == s.steps) {
        Pack<float, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; v++) o.v[v] = h[v];
        store<float, VEC>(lane_of(s.last + row0, c.at), o);
    }
}

// Backward. PART: the composites of all segments but the first alone, for C: from the end of a segment to its
// beginning, which need the gate and dh.
template <class T, int VEC, bool PART>
__global__ __launch_bounds__(64 * SCAN_WAVES, VEC <= 2 ? 4 : 2) void k_scan_bwd(const Scan s) {
    constexpr int STEPS = SCAN_STEPS;
    __shared__ Exchange<VEC> ex[2][3];
    __shared__ uint32_t flags[2][SCAN_WAVES];
    const Cells<VEC> c = cells_of<VEC>(s, unit_of(s));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    const int segment = blockIdx.y + (PART ? 1 : 0);
    const int64_t begin = (int64_t)segment * s.seg, end = begin + s.seg < s.steps ? begin + s.seg : s.steps;
    const T *x = (const T *)s.x + c.row * s.x_n, *gate = (const T *)s.gate + c.row * s.gate_n, *dh = (const T *)s.dh + c.row * s.dh_n;
    T *dx = (T *)s.dx + c.row * s.dx_n, *dg = (T *)s.dgate + c.row * s.dgate_n;
    const int64_t row0 = c.row * s.width;
    float A[VEC], C[VEC];
    int turn = 0;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        A[v] = 1.f;
        C[v] = PART ? 0.f : s.dlast ? s.dlast[row0 + c.at + v] : 0.f;
    }
    if (!PART && segment < s.segments - 1) {      // what the segments behind hand over
        const int n = s.segments - 1 - segment, per = (n + waves - 1) / waves, lo = wave * per < n ? wave * per : n,
                  hi = lo + per < n ? lo + per : n;
        float a[VEC], b[VEC];
        join<VEC>(s, row0, c.at, lo, hi, [&](int k) { return s.segments - 1 - k; }, a, b);
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[0][0].v[wave][v][lane] = a[v];
            ex[0][1].v[wave][v][lane] = b[v];
        }
        __syncthreads();
        for (int w = 0; w < waves; w++)
#pragma unroll
            for (int v = 0; v < VEC; v++) C[v] = after(ex[0][0].v[w][v][lane], ex[0][1].v[w][v][lane], C[v]);
        turn = 1;
    }
    const int span = waves * STEPS;
    for (int64_t tile = begin + (end - 1 - begin) / span * span; tile >= begin; tile -= span, turn ^= 1) {
        const int64_t first = tile + wave * STEPS;
        float a[STEPS][VEC], z[STEPS][VEC], e[STEPS][VEC], ca[VEC], cb[VEC], cr[VEC], h[VEC];
        Pack<T, VEC> px[STEPS], pg[STEPS], pd[STEPS];
        uint32_t drop = 0;
#pragma unroll
        for (int v = 0; v < VEC; v++) ca[v] = 1.f, cb[v] = 0.f, cr[v] = 0.f, h[v] = 0.f;
        if (!PART) {
            const float *before = tile ? s.marks + (tile / MARK - 1) * s.cells : s.state;
            if (before) {
                const Pack<float, VEC> m = load<float, VEC>(lane_of(before + row0, c.at));
#pragma unroll
                for (int v = 0; v < VEC; v++) h[v] = m.v[v];
            }
        }
        if (first < end) {
            rows_of<STEPS, T, VEC>(gate, s.gate_t, c.at, first, end, pg);
            if (!PART) rows_of<STEPS, T, VEC>(x, s.x_t, c.at, first, end, px);
            rows_of<STEPS, T, VEC>(dh, s.dh_t, c.at, first, end, pd);
            drop = resets_of<STEPS>(s, c.row, first, end);
            if (first + STEPS > end) {        // steps past the end change nothing: z = 0, a = 1
#pragma unroll
                for (int j = 0; j < STEPS; j++)
                    if (first + j >= end)
#pragma unroll
                        for (int v = 0; v < VEC; v++) {
                            pg[j].v[v] = (T)-INFINITY;
                            px[j].v[v] = pd[j].v[v] = (T)0.f;
                        }
            }
#pragma unroll
            for (int j = 0; j < STEPS; j++)
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const bool cut = drop >> j & 1;
                    gate_of<T>((float)pg[j].v[v], z[j][v], a[j][v]);
                    if (!PART) cb[v] = __builtin_fmaf(a[j][v], cut ? 0.f : cb[v], z[j][v] * (float)px[j].v[v]);
                    ca[v] = cut ? -1.f : ca[v] * a[j][v];
                }
#pragma unroll
            for (int j = STEPS - 1; j >= 0; j--)
#pragma unroll
                for (int v = 0; v < VEC; v++) cr[v] = drop >> j & 1 ? 0.f : a[j][v] * ((float)pd[j].v[v] + cr[v]);
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[turn][0].v[wave][v][lane] = ca[v];
            ex[turn][1].v[wave][v][lane] = cr[v];
            if (!PART) ex[turn][2].v[wave][v][lane] = cb[v];
        }
        if (lane == 0) flags[turn][wave] = drop;
        __syncthreads();
        const bool some = flags_of(flags[turn], waves) != 0;
        float mine[VEC];
        for (int w = waves - 1; w >= 0; w--) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                if (w == wave) mine[v] = C[v];
                const float pa = ex[turn][0].v[w][v][lane], pr = ex[turn][1].v[w][v][lane];
                C[v] = past_wave(pa, pr, C[v], some);
                if (PART) A[v] = __float_as_int(pa) < 0 ? -1.f : A[v] * pa;
            }
        }
        if (!PART && first < end) {
            for (int w = 0; w < wave; w++)
#pragma unroll
                for (int v = 0; v < VEC; v++) h[v] = past_wave(ex[turn][0].v[w][v][lane], ex[turn][2].v[w][v][lane], h[v], some);
#pragma unroll
            for (int j = 0; j < STEPS; j++)
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const float in = (float)px[j].v[v], before = drop >> j & 1 ? 0.f : h[v];
                    e[j][v] = (in - before) * (z[j][v] * a[j][v]);
                    h[v] = __builtin_fmaf(a[j][v], before, z[j][v] * in);
                }
            if (c.any)
#pragma unroll
                for (int j = STEPS - 1; j >= 0; j--) {
                    Pack<T, VEC> ox, og;
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        const float g = (float)pd[j].v[v] + mine[v];
                        ox.v[v] = (T)(z[j][v] * g);
                        og.v[v] = (T)(g * e[j][v]);
                        mine[v] = drop >> j & 1 ? 0.f : a[j][v] * g;
                    }
                    if (first + j < end) {
                        put_row<T, VEC>(lane_of(dx + (first + j) * s.dx_t, c.at), ox, s.past);
                        put_row<T, VEC>(lane_of(dg + (first + j) * s.dgate_t, c.at), og, s.past);
                    }
                }
        }
    }
    if (wave || !c.any) return;
    if (PART) {
        Pack<float, VEC> pa, pb;
#pragma unroll
        for (int v = 0; v < VEC; v++) pa.v[v] = A[v], pb.v[v] = C[v];
        store<float, VEC>(lane_of(s.parts + segment * s.cells + row0, c.at), pa);
        store<float, VEC>(lane_of(s.parts + (s.segments + segment) * s.cells + row0, c.at), pb);
    } else if (s.dstate && segment == 0) {
        Pack<float, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; v++) o.v[v] = C[v];
        store<float, VEC>(lane_of(s.dstate + row0, c.at), o);
    }
}

struct ScanCut {
    int vec, steps, columns, segments, seg;      // steps: of a wave at a time
    bool own;                                    // each wave alone
};
// What a pass costs a lane's place with 1, 2 or 4 channels a lane, in hundredths, on full lanes. 128 x 8,192 x 256 bf16:
// forward 458, 362 and 357 us, backward 715, 625 and 843 (four channels take the registers of a second workgroup on a CU);
// 250 x 500 x 256 fp32 61, 62 and 65, 140, 136 and 138; a single step of 65,536 x 256 bf16 52, 43 and 35, 71, 62 and 48.
inline int scan_cost(int vec, bool own, bool bwd, int type) {
    static const int alone[3] = {150, 122, 100}, fwd16[3] = {128, 102, 100}, bwd16[3] = {114, 100, 135}, fwd32[3] = {100, 101, 106},
                     bwd32[3] = {103, 100, 101};
    const int at = vec == 4 ? 2 : vec - 1;
    return own ? alone[at] : type == D1_FP32 ? (bwd ? bwd32[at] : fwd32[at]) : bwd ? bwd16[at] : fwd16[at];
}
// Fewer channels a lane waste less of a row's last lanes (2,000 x 300 fp16 of 40 steps: forward 47, 40 and 65 us) and make more
// workgroups. A sequence is cut where the workgroups would be under one a CU; cutting reads inputs twice (a third
// more time), and needs segments of two MARKs or more (4,000 x 3 x 700 bf16, 31 of them: 1,023 workgroups 30 us, 279 44).
inline ScanCut scan_cut(int64_t steps, int64_t rows, int width, int type, bool bwd) {
    ScanCut c{};
    c.own = steps <= SCAN_STEPS;
    c.steps = steps == 1 ? 1 : steps <= 4 ? 4 : SCAN_STEPS;
    const int64_t marks = (steps + MARK - 1) / MARK;
    double least = 0.0;
    for (int vec : {1, 2, 4}) {
        if (vec > width) break;
        const int64_t columns = (width + 64 * vec - 1) / (64 * vec), groups = rows * columns;
        const bool cut = !c.own && groups < 256 && marks >= 4;
        if (vec > 1 && !c.own && (cut ? groups * (marks / 2) < 1000 : groups < 256)) break;
        const double cost = (double)columns * 64 * vec * scan_cost(vec, c.own, bwd, type) * (cut ? 1.33 : 1.0);
        if (c.vec && cost >= least) continue;
        least = cost;
        int64_t segments = cut ? (1024 + groups - 1) / groups : 1;
        if (segments > marks / 2) segments = marks / 2;
        if (segments < 1) segments = 1;
        const int64_t per = (marks + segments - 1) / segments;
        c.vec = vec;
        c.columns = (int)columns;
        c.segments = segments > 1 ? (int)((marks + per - 1) / per) : 1;
        c.seg = (int)((c.segments > 1 ? per : marks < 1 ? 1 : marks) * MARK);
    }
    return c;
}

static bool scan_args(const D1Scan *h) {
    if (!h || !is_type(h->type) || h->steps < 0 || h->rows < 0 || h->width < 0 || h->width > D1_SCAN_MAX_WIDTH ||
        h->steps > D1_SCAN_MAX_STEPS)
        return false;
    return h->rows <= ((int64_t)1 << 48) / (h->width > 0 ? h->width : 1);
}
static bool scan_fill(const D1Scan *h, Scan &s, ScanCut &c, bool bwd) {
    c = scan_cut(h->steps, h->rows, h->width, h->type, bwd);
    s.steps = h->steps;
    s.width = h->width;
    s.cells = h->rows * h->width;
    s.columns = c.columns;
    s.segments = c.segments;
    s.seg = c.seg;
    s.past = (double)h->steps * s.cells * (h->type == D1_FP32 ? 4 : 2) > PAST_BYTES;
    s.x = h->x;
    s.x_t = h->x_t;
    s.x_n = h->x_n;
    s.gate = h->gate;
    s.gate_t = h->gate_t;
    s.gate_n = h->gate_n;
    s.reset = h->reset;
    s.reset_t = h->reset_t;
    s.reset_n = h->reset_n;
    s.state = h->state;
    s.marks = h->marks;
    return h->x && h->gate;
}
template <bool BWD, class T, int VEC, int STEPS>
static void scan_alone(const Scan &s, hipStream_t stream) {
    if (BWD)
        hipLaunchKernelGGL((k_scan_own_bwd<T, VEC, STEPS>), dim3((s.units + 3) / 4), dim3(256), 0, stream, s);
    else
        hipLaunchKernelGGL((k_scan_own_fwd<T, VEC, STEPS>), dim3((s.units + 3) / 4), dim3(256), 0, stream, s);
}
template <bool BWD, class T, int VEC, bool PART>
static void scan_shared(const Scan &s, int segments, hipStream_t stream) {
    const int waves = s.steps >= MARK ? SCAN_WAVES : (int)((s.steps + SCAN_STEPS - 1) / SCAN_STEPS);
    if (BWD)
        hipLaunchKernelGGL((k_scan_bwd<T, VEC, PART>), dim3(s.units, segments), dim3(64 * waves), 0, stream, s);
    else
        hipLaunchKernelGGL((k_scan_fwd<T, VEC, PART>), dim3(s.units, segments), dim3(64 * waves), 0, stream, s);
}
template <bool BWD, class T, int VEC>
static int scan_kind(const Scan &s, const ScanCut &c, hipStream_t stream) {
    if (c.own) {
        if (c.steps == 1)
            scan_alone<BWD, T, VEC, 1>(s, stream);
        else if (c.steps == 4)
            scan_alone<BWD, T, VEC, 4>(s, stream);
        else
            scan_alone<BWD, T, VEC, SCAN_STEPS>(s, stream);
        return (int)hipGetLastError();
    }
    if (c.segments > 1) scan_shared<BWD, T, VEC, true>(s, c.segments - 1, stream);
    scan_shared<BWD, T, VEC, false>(s, c.segments, stream);
    return (int)hipGetLastError();
}
template <bool BWD, class T>
static int scan_vec(const Scan &s, const ScanCut &c, hipStream_t stream) {
    return c.vec == 4 ? scan_kind<BWD, T, 4>(s, c, stream) : c.vec == 2 ? scan_kind<BWD, T, 2>(s, c, stream) : scan_kind<BWD, T, 1>(s, c, stream);
}
// A launch takes 2^22 units at most (a grid has under 2^32 threads); what is the rows' own is moved on for the next.
constexpr int64_t LAUNCH_UNITS = (int64_t)1 << 22;
static Scan scan_from(const Scan &s, int64_t row, int64_t rows, int type) {
    Scan p = s;
    const int64_t size = type == D1_FP32 ? 4 : 2, cell = row * s.width;
    auto on = [&](auto *&at, int64_t bytes) {
        if (at) at = (std::remove_reference_t<decltype(at)>)((uintptr_t)at + bytes);
    };
    on(p.x, row * s.x_n * size);
    on(p.gate, row * s.gate_n * size);
    on(p.h, row * s.h_n * size);
    on(p.dh, row * s.dh_n * size);
    on(p.dx, row * s.dx_n * size);
    on(p.dgate, row * s.dgate_n * size);
    on(p.reset, row * s.reset_n);
    on(p.state, cell * 4);
    on(p.last, cell * 4);
    on(p.dlast, cell * 4);
    on(p.dstate, cell * 4);
    on(p.marks, cell * 4);
    on(p.parts, cell * 4);
    p.units = (uint32_t)(rows * s.columns);
    return p;
}
template <bool BWD>
static int scan_type(const Scan &s, const ScanCut &c, const D1Scan *h, hipStream_t stream) {
    const int64_t most = LAUNCH_UNITS / c.columns;            // columns: 2^18 at most
    for (int64_t row = 0; row < h->rows; row += most) {
        const Scan p = scan_from(s, row, h->rows - row < most ? h->rows - row : most, h->type);
        const int code = h->type == D1_FP32 ? scan_vec<BWD, float>(p, c, stream)
                         : h->type == D1_BF16 ? scan_vec<BWD, __bf16>(p, c, stream) : scan_vec<BWD, _Float16>(p, c, stream);
        if (code) return code;
    }
    return 0;
}

}  // namespace d1o

using namespace d1o;

extern "C" {
int64_t d1_scan_marks(const D1Scan *h) {
    if (!scan_args(h)) return D1_E_ARG;
    return h->steps > MARK ? (h->steps + MARK - 1) / MARK - 1 : 0;
}

int64_t d1_scan_work_bytes(const D1Scan *h) {
    if (!scan_args(h)) return D1_E_ARG;
    if (h->steps == 0 || h->rows == 0 || h->width == 0) return 0;         // nothing to cut
    const int f = scan_cut(h->steps, h->rows, h->width, h->type, false).segments, b = scan_cut(h->steps, h->rows, h->width, h->type, true).segments;
    const int most = f > b ? f : b;
    return most > 1 ? (int64_t)2 * sizeof(float) * most * h->rows * h->width : 0;
}

int d1_scan_fwd(const D1Scan *h, void *out, int64_t out_t, int64_t out_n, float *last, void *work, int64_t work_bytes, void *stream) {
    if (!scan_args(h)) return D1_E_ARG;
    if (h->steps == 0 || h->rows == 0 || h->width == 0) return 0;
    Scan s{};
    ScanCut c;
    if (!scan_fill(h, s, c, false) || !out) return D1_E_ARG;
    const int64_t need = d1_scan_work_bytes(h);
    if (need && (!work || work_bytes < need || ((uintptr_t)work & 3))) return D1_E_ARG;
    s.h = out;
    s.h_t = out_t;
    s.h_n = out_n;
    s.last = last;
    s.parts = (float *)work;
    return scan_type<false>(s, c, h, (hipStream_t)stream);
}

int d1_scan_bwd(const D1Scan *h, const void *dh, int64_t dh_t, int64_t dh_n, const float *dlast, void *dx, int64_t dx_t, int64_t dx_n,
                void *dgate, int64_t dgate_t, int64_t dgate_n, float *dstate, void *work, int64_t work_bytes, void *stream) {
    if (!scan_args(h)) return D1_E_ARG;
    if (h->steps == 0 || h->rows == 0 || h->width == 0) return 0;
    Scan s{};
    ScanCut c;
    if (!scan_fill(h, s, c, true) || !dh || !dx || !dgate || (d1_scan_marks(h) && !h->marks)) return D1_E_ARG;
    const int64_t need = d1_scan_work_bytes(h);
    if (need && (!work || work_bytes < need || ((uintptr_t)work & 3))) return D1_E_ARG;
    s.dh = dh;
    s.dh_t = dh_t;
    s.dh_n = dh_n;
    s.dlast = dlast;
    s.dx = dx;
    s.dx_t = dx_t;
    s.dx_n = dx_n;
    s.dgate = dgate;
    s.dgate_t = dgate_t;
    s.dgate_n = dgate_n;
    s.dstate = dstate;
    s.parts = (float *)work;
    return scan_type<true>(s, c, h, (hipStream_t)stream);
}
}
