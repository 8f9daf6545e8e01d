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
// workgroup goes on along its sequence, so every input is read once. Where channels alone would leave CUs idle, the
// sequence is cut into segments: a first launch forms the segments' composites and the second starts each segment from
// those before it (no workgroup waits for another). The backward pass reads no h: forward keeps the fp32 state before
// every MARK-th step and the backward pass makes the states between again, which costs 4 bytes a channel in MARK steps
// and gives dgate from states that were never rounded to 16 bits.
// A product A is -1 (sign bit) once a reset lies in it: what comes before is dropped, even where it is not finite.
// Everything is computed in fp32.
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
    int32_t width, columns;               // columns: workgroups beside each other on one row's channels
    int32_t segments, seg;                // seg: steps of a segment, a multiple of MARK
};

template <int VEC>
struct Cells {
    int64_t row;
    int32_t at;                           // first channel of the lane
    bool mine;                            // not one that other lanes hold too
    bool any;
};
// the lane's channels; those past the end are moved back over it (both lanes then store the same values)
template <int VEC>
__device__ __forceinline__ Cells<VEC> cells_of(const Scan &s) {
    Cells<VEC> c;
    c.row = blockIdx.x / s.columns;
    const int at = ((int)(blockIdx.x % s.columns) * 64 + (threadIdx.x & 63)) * VEC;
    c.any = at < s.width;
    c.at = at < s.width - VEC ? at : s.width - VEC;
    return c;
}

// z = sigmoid(g) and a = sigmoid(-g), each exact to a few ulp where it is small too. e^-|g| is 2^p of the rounded product
// p = -|g| log2 e, times what the rounding dropped.
__device__ __forceinline__ void gate_of(float g, float &z, float &a) {
    const float y = -fminf(fabsf(g), 104.f), p = y * 1.44269504f;
    const float rest = __builtin_fmaf(y, 1.44269504f, -p) + y * 1.92596299e-8f;
    float e = __builtin_amdgcn_exp2f(p);
    e = __builtin_fmaf(e, rest * 0.693147181f, e);
    const float big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
    z = g >= 0.f ? big : small;
    a = g >= 0.f ? small : big;
    if (g != g) z = a = g;
}

// the bits of the steps that drop what was before: step first + j in bit j
__device__ __forceinline__ uint32_t resets_of(const Scan &s, int64_t row, int64_t first, int64_t end) {
    if (!s.reset) return 0;
    const int j = threadIdx.x & 63;
    const bool r = j < SCAN_STEPS && first + j < end && s.reset[(first + j) * s.reset_t + row * s.reset_n];
    return (uint32_t)__ballot(r);
}

// the state after the composite (a, b)
__device__ __forceinline__ float after(float a, float b, float h) { return __float_as_int(a) < 0 ? b : __builtin_fmaf(a, h, b); }

template <class T, int VEC>
__device__ __forceinline__ void rows_of(const T *p, int64_t st, int64_t first, int64_t end, Pack<T, VEC> *out) {
#pragma unroll
    for (int j = 0; j < SCAN_STEPS; j++) {
        const int64_t t = first + j < end ? first + j : end - 1;
        out[j] = load<T, VEC>(p + t * st);
    }
}

// Forward. PART: the composites of all segments but the last alone.
template <class T, int VEC, bool PART>
__global__ __launch_bounds__(64 * SCAN_WAVES) void k_scan_fwd(const Scan s) {
    __shared__ float ex[2][2][SCAN_WAVES][VEC][64];
    const Cells<VEC> c = cells_of<VEC>(s);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    const int64_t begin = (int64_t)blockIdx.y * s.seg, end = begin + s.seg < s.steps ? begin + s.seg : s.steps;
    const T *x = (const T *)s.x + c.row * s.x_n + c.at, *gate = (const T *)s.gate + c.row * s.gate_n + c.at;
    const int64_t cell = c.row * s.width + c.at;
    float A[VEC], h[VEC];                 // the workgroup's composite so far (PART), or the state
    int turn = 0;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        A[v] = 1.f;
        h[v] = PART ? 0.f : s.state ? s.state[cell + v] : 0.f;
    }
    if (!PART && blockIdx.y) {            // the state that the segments before leave: each wave joins a share of them
        const int n = blockIdx.y, per = (n + waves - 1) / waves, lo = wave * per < n ? wave * per : n, hi = lo + per < n ? lo + per : n;
        float a[VEC], b[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) a[v] = 1.f, b[v] = 0.f;
        for (int k = lo; k < hi; k++) {
            const Pack<float, VEC> pa = load<float, VEC>(s.parts + k * s.cells + cell);
            const Pack<float, VEC> pb = load<float, VEC>(s.parts + (s.segments + k) * s.cells + cell);
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                b[v] = after(pa.v[v], pb.v[v], b[v]);
                a[v] = __float_as_int(pa.v[v]) < 0 ? -1.f : a[v] * pa.v[v];
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[0][0][wave][v][lane] = a[v];
            ex[0][1][wave][v][lane] = b[v];
        }
        __syncthreads();
        for (int w = 0; w < waves; w++)
#pragma unroll
            for (int v = 0; v < VEC; v++) h[v] = after(ex[0][0][w][v][lane], ex[0][1][w][v][lane], h[v]);
        turn = 1;
    }
    for (int64_t tile = begin; tile < end; tile += waves * SCAN_STEPS, turn ^= 1) {
        const int64_t first = tile + wave * SCAN_STEPS;
        float a[SCAN_STEPS][VEC], b[SCAN_STEPS][VEC], ca[VEC], cb[VEC];
        uint32_t drop = 0;
#pragma unroll
        for (int v = 0; v < VEC; v++) ca[v] = 1.f, cb[v] = 0.f;
        if (first < end) {
            Pack<T, VEC> px[SCAN_STEPS], pg[SCAN_STEPS];
            rows_of<T, VEC>(gate, s.gate_t, first, end, pg);
            rows_of<T, VEC>(x, s.x_t, first, end, px);
            drop = resets_of(s, c.row, first, end);
#pragma unroll
            for (int j = 0; j < SCAN_STEPS; j++) {
                const bool on = first + j < end;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    float z, k;
                    gate_of((float)pg[j].v[v], z, k);
                    a[j][v] = on ? k : 1.f;
                    b[j][v] = on ? z * (float)px[j].v[v] : 0.f;
                    if (drop >> j & 1) {
                        ca[v] = -1.f;
                        cb[v] = b[j][v];
                    } else {
                        ca[v] *= a[j][v];
                        cb[v] = __builtin_fmaf(a[j][v], cb[v], b[j][v]);
                    }
                }
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[turn][0][wave][v][lane] = ca[v];
            ex[turn][1][wave][v][lane] = cb[v];
        }
        __syncthreads();
        if (!PART && s.marks && tile % MARK == 0 && tile && wave == 0 && c.any) {
            Pack<float, VEC> m;
#pragma unroll
            for (int v = 0; v < VEC; v++) m.v[v] = h[v];
            store<float, VEC>(s.marks + (tile / MARK - 1) * s.cells + cell, m);
        }
        float mine[VEC];
        for (int w = 0; w < waves; w++) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                if (w == wave) mine[v] = h[v];
                const float pa = ex[turn][0][w][v][lane], pb = ex[turn][1][w][v][lane];
                h[v] = after(pa, pb, h[v]);
                if (PART) A[v] = __float_as_int(pa) < 0 ? -1.f : A[v] * pa;
            }
        }
        if (!PART && first < end && c.any) {
            T *out = (T *)s.h + c.row * s.h_n + c.at;
#pragma unroll
            for (int j = 0; j < SCAN_STEPS; j++) {
                if (first + j >= end) break;
                Pack<T, VEC> o;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    mine[v] = drop >> j & 1 ? b[j][v] : __builtin_fmaf(a[j][v], mine[v], b[j][v]);
                    o.v[v] = (T)mine[v];
                }
                store<T, VEC>(out + (first + j) * s.h_t, o);
            }
        }
    }
    if (wave || !c.any) return;
    if (PART) {
        Pack<float, VEC> pa, pb;
#pragma unroll
        for (int v = 0; v < VEC; v++) pa.v[v] = A[v], pb.v[v] = h[v];
        store<float, VEC>(s.parts + blockIdx.y * s.cells + cell, pa);
        store<float, VEC>(s.parts + (s.segments + blockIdx.y) * s.cells + cell, pb);
    } else if (s.last && end == s.steps) {
        Pack<float, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; v++) o.v[v] = h[v];
        store<float, VEC>(s.last + cell, o);
    }
}

// Backward. PART: the composites of all segments but the first alone, for C: from the end of a segment to its
// beginning, which need the gate and dh.
template <class T, int VEC, bool PART>
__global__ __launch_bounds__(64 * SCAN_WAVES) void k_scan_bwd(const Scan s) {
    __shared__ float ex[2][3][SCAN_WAVES][VEC][64];
    const Cells<VEC> c = cells_of<VEC>(s);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    const int segment = blockIdx.y + (PART ? 1 : 0);
    const int64_t begin = (int64_t)segment * s.seg, end = begin + s.seg < s.steps ? begin + s.seg : s.steps;
    const T *x = (const T *)s.x + c.row * s.x_n + c.at, *gate = (const T *)s.gate + c.row * s.gate_n + c.at;
    const T *dh = (const T *)s.dh + c.row * s.dh_n + c.at;
    const int64_t cell = c.row * s.width + c.at;
    float A[VEC], C[VEC];
    int turn = 0;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        A[v] = 1.f;
        C[v] = PART ? 0.f : s.dlast ? s.dlast[cell + v] : 0.f;
    }
    if (!PART && segment < s.segments - 1) {      // what the segments behind hand over
        const int n = s.segments - 1 - segment, per = (n + waves - 1) / waves, lo = wave * per < n ? wave * per : n,
                  hi = lo + per < n ? lo + per : n;
        float a[VEC], b[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) a[v] = 1.f, b[v] = 0.f;
        for (int k = lo; k < hi; k++) {
            const int from = s.segments - 1 - k;
            const Pack<float, VEC> pa = load<float, VEC>(s.parts + from * s.cells + cell);
            const Pack<float, VEC> pb = load<float, VEC>(s.parts + (s.segments + from) * s.cells + cell);
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                b[v] = after(pa.v[v], pb.v[v], b[v]);
                a[v] = __float_as_int(pa.v[v]) < 0 ? -1.f : a[v] * pa.v[v];
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[0][0][wave][v][lane] = a[v];
            ex[0][1][wave][v][lane] = b[v];
        }
        __syncthreads();
        for (int w = 0; w < waves; w++)
#pragma unroll
            for (int v = 0; v < VEC; v++) C[v] = after(ex[0][0][w][v][lane], ex[0][1][w][v][lane], C[v]);
        turn = 1;
    }
    const int span = waves * SCAN_STEPS;
    for (int64_t tile = begin + (end - 1 - begin) / span * span; tile >= begin; tile -= span, turn ^= 1) {
        const int64_t first = tile + wave * SCAN_STEPS;
        // a, the slope z a (x - m h[t-1]) as it becomes known, dh, z
        float a[SCAN_STEPS][VEC], z[SCAN_STEPS][VEC], e[SCAN_STEPS][VEC], d[SCAN_STEPS][VEC], ca[VEC], cb[VEC], cr[VEC], h[VEC];
        uint32_t drop = 0;
#pragma unroll
        for (int v = 0; v < VEC; v++) ca[v] = 1.f, cb[v] = 0.f, cr[v] = 0.f, h[v] = 0.f;
        if (!PART) {
            const float *before = tile ? s.marks + (tile / MARK - 1) * s.cells : s.state;
            if (before) {
                const Pack<float, VEC> m = load<float, VEC>(before + cell);
#pragma unroll
                for (int v = 0; v < VEC; v++) h[v] = m.v[v];
            }
        }
        if (first < end) {
            Pack<T, VEC> px[SCAN_STEPS], pg[SCAN_STEPS], pd[SCAN_STEPS];
            rows_of<T, VEC>(gate, s.gate_t, first, end, pg);
            if (!PART) rows_of<T, VEC>(x, s.x_t, first, end, px);
            rows_of<T, VEC>(dh, s.dh_t, first, end, pd);
            drop = resets_of(s, c.row, first, end);
#pragma unroll
            for (int j = 0; j < SCAN_STEPS; j++) {
                const bool on = first + j < end;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    float k;
                    gate_of((float)pg[j].v[v], z[j][v], k);
                    a[j][v] = on ? k : 1.f;
                    d[j][v] = on ? (float)pd[j].v[v] : 0.f;
                    if (!PART) {
                        e[j][v] = on ? (float)px[j].v[v] : 0.f;
                        const float b = on ? z[j][v] * e[j][v] : 0.f;
                        cb[v] = drop >> j & 1 ? b : __builtin_fmaf(a[j][v], cb[v], b);
                    }
                    ca[v] = drop >> j & 1 ? -1.f : ca[v] * a[j][v];
                }
            }
#pragma unroll
            for (int j = SCAN_STEPS - 1; j >= 0; j--)
#pragma unroll
                for (int v = 0; v < VEC; v++) cr[v] = drop >> j & 1 ? 0.f : a[j][v] * (d[j][v] + cr[v]);
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            ex[turn][0][wave][v][lane] = ca[v];
            ex[turn][1][wave][v][lane] = cr[v];
            if (!PART) ex[turn][2][wave][v][lane] = cb[v];
        }
        __syncthreads();
        float mine[VEC];
        for (int w = waves - 1; w >= 0; w--) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                if (w == wave) mine[v] = C[v];
                const float pa = ex[turn][0][w][v][lane], pr = ex[turn][1][w][v][lane];
                C[v] = after(pa, pr, C[v]);
                if (PART) A[v] = __float_as_int(pa) < 0 ? -1.f : A[v] * pa;
            }
        }
        if (!PART && first < end) {
            for (int w = 0; w < wave; w++)
#pragma unroll
                for (int v = 0; v < VEC; v++) h[v] = after(ex[turn][0][w][v][lane], ex[turn][2][w][v][lane], h[v]);
#pragma unroll
            for (int j = 0; j < SCAN_STEPS; j++)
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const float x_ = e[j][v], before = drop >> j & 1 ? 0.f : h[v];
                    e[j][v] = (x_ - before) * (z[j][v] * a[j][v]);
                    h[v] = __builtin_fmaf(a[j][v], before, z[j][v] * x_);
                }
            if (c.any) {
                T *dx = (T *)s.dx + c.row * s.dx_n + c.at, *dg = (T *)s.dgate + c.row * s.dgate_n + c.at;
#pragma unroll
                for (int j = SCAN_STEPS - 1; j >= 0; j--) {
                    Pack<T, VEC> ox, og;
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        const float g = d[j][v] + mine[v];
                        ox.v[v] = (T)(z[j][v] * g);
                        og.v[v] = (T)(g * e[j][v]);
                        mine[v] = drop >> j & 1 ? 0.f : a[j][v] * g;
                    }
                    if (first + j < end) {
                        store<T, VEC>(dx + (first + j) * s.dx_t, ox);
                        store<T, VEC>(dg + (first + j) * s.dgate_t, og);
                    }
                }
            }
        }
    }
    if (wave || !c.any) return;
    if (PART) {
        Pack<float, VEC> pa, pb;
#pragma unroll
        for (int v = 0; v < VEC; v++) pa.v[v] = A[v], pb.v[v] = C[v];
        store<float, VEC>(s.parts + segment * s.cells + cell, pa);
        store<float, VEC>(s.parts + (s.segments + segment) * s.cells + cell, pb);
    } else if (s.dstate && segment == 0) {
        Pack<float, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; v++) o.v[v] = C[v];
        store<float, VEC>(s.dstate + cell, o);
    }
}

struct ScanCut {
    int vec, waves, columns, segments, seg;
};
// One wave for up to SCAN_STEPS steps, up to SCAN_WAVES behind each other; four channels a lane where a row has 256,
// one where it has 64 or fewer. A sequence is cut into segments where the workgroups would be under two a CU.
inline ScanCut scan_cut(int64_t steps, int64_t rows, int width) {
    ScanCut c;
    c.vec = width >= 192 ? 4 : width >= 96 ? 2 : 1;
    c.columns = (width + 64 * c.vec - 1) / (64 * c.vec);
    c.waves = steps >= MARK ? SCAN_WAVES : (int)((steps + SCAN_STEPS - 1) / SCAN_STEPS);
    const int64_t groups = rows * c.columns, marks = (steps + MARK - 1) / MARK;
    int64_t cut = groups >= 512 || marks < 4 ? 1 : (1024 + groups - 1) / groups;
    if (cut > marks / 2) cut = marks / 2;
    if (cut < 1) cut = 1;
    const int64_t per = (marks + cut - 1) / cut;
    c.seg = (int)(cut == 1 ? (marks < 1 ? 1 : marks) * MARK : per * MARK);
    c.segments = cut == 1 ? 1 : (int)((marks + per - 1) / per);
    return c;
}

static bool scan_args(const D1Scan *h) {
    if (!h || !is_type(h->type) || h->steps < 0 || h->rows < 0 || h->width < 0 || h->width > D1_SCAN_MAX_WIDTH ||
        h->steps > D1_SCAN_MAX_STEPS)
        return false;
    const int64_t columns = (h->width + 63) / 64;
    return h->rows <= (int64_t)0x7FFFFFFF / (columns > 0 ? columns : 1);
}
static bool scan_fill(const D1Scan *h, Scan &s, ScanCut &c) {
    c = scan_cut(h->steps, h->rows, h->width);
    s.steps = h->steps;
    s.width = h->width;
    s.cells = h->rows * h->width;
    s.columns = c.columns;
    s.segments = c.segments;
    s.seg = c.seg;
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
template <bool BWD, class T, int VEC>
static int scan_launch(const Scan &s, const ScanCut &c, int64_t rows, hipStream_t stream) {
    const dim3 block(64 * c.waves);
    const unsigned groups = (unsigned)(rows * c.columns);
    if (c.segments > 1) {
        if (BWD)
            hipLaunchKernelGGL((k_scan_bwd<T, VEC, true>), dim3(groups, c.segments - 1), block, 0, stream, s);
        else
            hipLaunchKernelGGL((k_scan_fwd<T, VEC, true>), dim3(groups, c.segments - 1), block, 0, stream, s);
    }
    if (BWD)
        hipLaunchKernelGGL((k_scan_bwd<T, VEC, false>), dim3(groups, c.segments), block, 0, stream, s);
    else
        hipLaunchKernelGGL((k_scan_fwd<T, VEC, false>), dim3(groups, c.segments), block, 0, stream, s);
    return (int)hipGetLastError();
}
template <bool BWD, class T>
static int scan_vec(const Scan &s, const ScanCut &c, int64_t rows, hipStream_t stream) {
    return c.vec == 4 ? scan_launch<BWD, T, 4>(s, c, rows, stream) : c.vec == 2 ? scan_launch<BWD, T, 2>(s, c, rows, stream)
                                                                                : scan_launch<BWD, T, 1>(s, c, rows, stream);
}
template <bool BWD>
static int scan_type(const Scan &s, const ScanCut &c, const D1Scan *h, hipStream_t stream) {
    return h->type == D1_FP32 ? scan_vec<BWD, float>(s, c, h->rows, stream)
           : h->type == D1_BF16 ? scan_vec<BWD, __bf16>(s, c, h->rows, stream) : scan_vec<BWD, _Float16>(s, c, h->rows, stream);
}

}  // namespace d1o

using namespace d1o;

extern "C" {
int64_t d1_scan_marks(int64_t steps) { return steps > MARK ? (steps + MARK - 1) / MARK - 1 : 0; }

int64_t d1_scan_work_bytes(const D1Scan *h) {
    if (!scan_args(h)) return D1_E_ARG;
    const ScanCut c = scan_cut(h->steps, h->rows, h->width);
    return c.segments > 1 ? (int64_t)2 * sizeof(float) * c.segments * h->rows * h->width : 0;
}

int d1_scan_fwd(const D1Scan *h, void *out, int64_t out_t, int64_t out_n, float *last, void *work, int64_t work_bytes, void *stream) {
    if (!scan_args(h)) return D1_E_ARG;
    if (h->steps == 0 || h->rows == 0 || h->width == 0) return 0;
    Scan s{};
    ScanCut c;
    if (!scan_fill(h, s, c) || !out) return D1_E_ARG;
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
    if (!scan_fill(h, s, c) || !dh || !dx || !dgate || (d1_scan_marks(h->steps) && !h->marks)) return D1_E_ARG;
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
