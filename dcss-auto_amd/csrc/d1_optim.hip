// d1ops: one AdamW step over many tensors, moments in 32 or 8 bits, gfx950.
//
//   g' = c g;  m = b1 m + (1-b1) g';  v = b2 v + (1-b2) g'^2
//   p = p (1 - lr wd) - (lr / (1-b1^t)) m / (sqrt(v) / sqrt(1-b2^t) + eps)
// A launch carries the addresses of up to MAX_TENSORS tensors in its arguments (nothing is uploaded);
// a workgroup of 256 takes CHUNK adjacent elements of one of them, four at a time a lane, so each
// operand is one 16-byte access. k_adamw_begin, one workgroup before the step, advances the step
// count on the device, forms the two bias corrections in fp64 and, for a clip, adds the partial
// sums of squares of k_adamw_norm (fp64, a fixed order: the same bits each time). Up to JOIN_PARTS
// partial sums are added by each of the step's workgroups instead, one launch less: the policy's
// 0.53 M elements 10.9 -> 9.7 us, 1 M 12.5 and 12.2, but 4.2 M (2,048 sums) 29.1 and 31.2.
//
// 8-bit moments. 256 adjacent elements (a wave's four a lane) share one power of two, the exponent
// e of their largest magnitude. An element is scaled by 2^(top-e) so that its fp32 exponent field
// is at most `top` (15 for m, 31 for v): the field and 3 bits of mantissa are the code, and what
// lies below the field's range is an fp32 denormal, which is the code's own linear range. Rounding
// adds a 16-bit draw below the code's last bit and cuts. Its expectation is the value: a moment that
// moves by less than a step an update (v moves by a thousandth, a step is an eighth) still follows
// its mean, where rounding to the nearest would leave it where it is.
// An element whose m or v is infinite (without a clip nothing keeps such a gradient out, nor one whose square overflows)
// does not count for the block's largest, which would put the 255 others below their codes' range; it starts anew
// from m = 0 and the largest v that its block's codes hold. A NaN, which no maximum takes in, becomes a block's largest code
// too; the parameter is NaN by then.
#include "d1_rows.h"

namespace d1o {

constexpr int CHUNK = 4096, SMALL_CHUNK = 1024, MAX_TENSORS = 40, NORM_GRID = 2048, JOIN_PARTS = 1024;
// of ctl
constexpr int STEP = 0, SKIPPED = 1, COEF = 2, INV_BC1 = 3, INV_BC2 = 4, NORM = 5, GO = 6, BEFORE = 7;

struct Tensors {
    void *p[MAX_TENSORS];
    const void *g[MAX_TENSORS];
    void *m[MAX_TENSORS], *v[MAX_TENSORS];
    uint8_t *m_exp[MAX_TENSORS], *v_exp[MAX_TENSORS];
    void *copy[MAX_TENSORS];
    int64_t n[MAX_TENSORS], counter[MAX_TENSORS];
    float lr[MAX_TENSORS], keep[MAX_TENSORS];            // keep = 1 - lr wd
    int32_t lag[MAX_TENSORS], last_chunk[MAX_TENSORS];   // last_chunk: chunks of this and all tensors before
    uint8_t types[MAX_TENSORS];                          // bit 0: p is bf16, bit 1: g is bf16
    int32_t count, chunks, chunk;                        // chunk: elements of one, CHUNK or SMALL_CHUNK
};
struct Rates {
    float b1, omb1, b2, omb2, eps;                       // omb = 1 - b
    double log_b1, log_b2;
    uint64_t seed;
};
// The gradients' partial sums of squares where the step's workgroups add them themselves (nullptr: k_adamw_begin has).
// `first`: workgroup 0 of this launch writes the new step count, the skips and the norm.
struct Join {
    const double *parts;
    int32_t count, first;
    double max_norm;
};

__device__ __forceinline__ void corrections(double log_b1, double log_b2, int step, float &inv1, float &inv2) {
    inv1 = (float)(1.0 / -expm1((double)step * log_b1));
    inv2 = (float)(1.0 / sqrt(-expm1((double)step * log_b2)));
}
// the factor of a clip; false for a norm that is not finite
__device__ __forceinline__ bool clip_of(double norm, double max_norm, double &coef) {
    coef = max_norm / (norm + 1e-6);
    if (!(coef < 1.0)) coef = 1.0;
    return isfinite(norm);
}

// the tensor of a chunk, and the chunk's number within it
__device__ __forceinline__ int tensor_of(const Tensors &t, int chunk, int &within) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (chunk < t.last_chunk[mid])
            hi = mid;
        else
            lo = mid + 1;
    }
    within = chunk - (lo ? t.last_chunk[lo - 1] : 0);
    return lo;
}

template <class T>
__device__ __forceinline__ void add_squares(double &sum, const T *g, int64_t begin, int64_t n, int chunk) {
    constexpr int VEC = 16 / (int)sizeof(T), ALL = CHUNK / 256 / VEC;
    const int64_t i = begin + threadIdx.x * VEC;
    Pack<T, VEC> a[ALL];
    if (chunk == CHUNK && begin + CHUNK <= n) {        // all loads before the first sum
#pragma unroll
        for (int u = 0; u < ALL; u++) a[u] = load<T, VEC>(g + i + u * 256 * VEC);
    } else {
        const int64_t end = begin + chunk < n ? begin + chunk : n;
#pragma unroll
        for (int u = 0; u < ALL; u++) {
            const int64_t left = end - (i + u * 256 * VEC);
            a[u] = load_part<T, VEC>(g + i + u * 256 * VEC, left > VEC ? VEC : left > 0 ? (int)left : 0, (T)0.f);
        }
    }
#pragma unroll
    for (int u = 0; u < ALL; u++)
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const double d = (double)(float)a[u].v[j];
            sum = __builtin_fma(d, d, sum);
        }
}

// partial sums of squares of the gradients: each workgroup walks `per` chunks in a row (369 M bf16 in two launches 138 us,
// 5.3 TB/s)
// For a step that joins them itself (`ctl`), workgroup 0 keeps the count before it and forms the bias corrections, since
// the step's workgroups read these while one of them writes the new count.
__global__ __launch_bounds__(256) void k_adamw_norm(const Tensors t, int per, double *__restrict__ parts, int32_t *__restrict__ ctl,
                                                    double log_b1, double log_b2) {
    __shared__ double s[256];
    double sum = 0.0;
    if (ctl && blockIdx.x == 0 && threadIdx.x == 255) {
        const int before = ctl[STEP];
        float inv1, inv2;
        corrections(log_b1, log_b2, before + 1, inv1, inv2);
        ctl[BEFORE] = before;
        ctl[INV_BC1] = __float_as_int(inv1);
        ctl[INV_BC2] = __float_as_int(inv2);
    }
    int chunk = blockIdx.x * per, within;
    const int end = chunk + per < t.chunks ? chunk + per : t.chunks;
    int k = tensor_of(t, chunk, within);
    for (; chunk < end; chunk++, within++) {
        if (chunk >= t.last_chunk[k]) {
            k++;
            within = 0;
        }
        const int64_t begin = (int64_t)within * t.chunk;
        if (t.types[k] & 2)
            add_squares(sum, (const __bf16 *)t.g[k], begin, t.n[k], t.chunk);
        else
            add_squares(sum, (const float *)t.g[k], begin, t.n[k], t.chunk);
    }
    s[threadIdx.x] = sum;
    __syncthreads();
    for (int d = 128; d; d >>= 1) {
        if ((int)threadIdx.x < d) s[threadIdx.x] += s[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) parts[blockIdx.x] = s[0];
}

__global__ __launch_bounds__(1024) void k_adamw_begin(int32_t *__restrict__ ctl, const double *__restrict__ parts, int nparts,
                                                      double max_norm, double log_b1, double log_b2) {
    __shared__ double s[1024];
    double coef = 1.0;
    bool go = true;
    if (parts) {
        double sum = 0.0;
        for (int i = threadIdx.x; i < nparts; i += 1024) sum += parts[i];
        s[threadIdx.x] = sum;
        __syncthreads();
        for (int d = 512; d; d >>= 1) {
            if ((int)threadIdx.x < d) s[threadIdx.x] += s[threadIdx.x + d];
            __syncthreads();
        }
        const double norm = sqrt(s[0]);
        go = clip_of(norm, max_norm, coef);
        if (threadIdx.x == 0) ctl[NORM] = __float_as_int((float)norm);
    }
    if (threadIdx.x) return;
    if (!parts && max_norm > 0.0) ctl[NORM] = 0;       // a clip of no elements
    ctl[GO] = go;
    if (!go) {
        ctl[SKIPPED]++;
        return;
    }
    const int step = ++ctl[STEP];
    float inv1, inv2;
    corrections(log_b1, log_b2, step, inv1, inv2);
    ctl[COEF] = __float_as_int((float)coef);
    ctl[INV_BC1] = __float_as_int(inv1);
    ctl[INV_BC2] = __float_as_int(inv2);
}

// ---- 8-bit moments

// a 32-bit word through two multiplications and three shifts
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x9E3779B1u;
    x ^= x >> 15;
    x *= 0xB7E15163u;
    return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t draw_key(uint64_t seed, uint32_t step, uint32_t counter_high) {
    return mix(mix(mix(mix((uint32_t)seed) ^ (uint32_t)(seed >> 32)) ^ step) ^ counter_high);
}
// the block's exponent field: one more where rounding up could pass the largest code
__device__ __forceinline__ int block_exp(float largest) { return (int)((__float_as_uint(largest) + 0xFFFFFu) >> 23); }
template <int TOP>
__device__ __forceinline__ uint32_t encode(float a, int e, uint32_t draw16) {
    const uint32_t c = (__float_as_uint(__builtin_ldexpf(a, TOP - e)) + (draw16 << 4)) >> 20;
    return c < (TOP + 1) * 8 ? c : (TOP + 1) * 8 - 1;
}
template <int TOP>
__device__ __forceinline__ float decode(uint32_t code, int e) {
    return __builtin_ldexpf(__uint_as_float((code & ((TOP + 1) * 8 - 1)) << 20), e - TOP);
}
__device__ __forceinline__ float decode_m(uint32_t code, int e) {
    const float a = decode<15>(code, e);
    return code & 128 ? -a : a;
}

// ---- the step

// m / (sqrt(v) inv + eps)
__device__ __forceinline__ float over32(float m, float v, float inv, float eps) { return m / (sqrtf(v) * inv + eps); }
// The same with the hardware's root and reciprocal (each within 1 ulp), for the 8-bit step, which is as much bound by its
// instructions as by memory: 369 M elements 1,265 -> 1,158 us (the 32-bit step gains nothing). The
// root has no denormal operands, so v is raised by 2^24; past 2^104 that overflows and the parameter stays.
__device__ __forceinline__ float over8(float m, float v, float inv, float eps) {
    return m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v * 0x1p24f) * (inv * 0x1p-12f) + eps);
}

template <class P, class G, int BITS, bool PAST>
__device__ __forceinline__ void step_chunk(const Tensors &t, int k, int within, const Rates &r, float coef, float inv1, float inv2,
                                           uint32_t step) {
    const int64_t n = t.n[k];
    const float size = t.lr[k] * inv1, keep = t.keep[k];
    P *p = (P *)t.p[k];
    const G *g = (const G *)t.g[k];
    __bf16 *copy = (__bf16 *)t.copy[k];
    for (int u = 0; u < t.chunk; u += 1024) {
        const int64_t first = (int64_t)within * t.chunk + u + (threadIdx.x & ~63u) * 4;         // of the wave's 256
        if (first >= n) return;                                                                 // the whole wave
        const int64_t i = first + (threadIdx.x & 63) * 4;
        const int have = n - i >= 4 ? 4 : n - i > 0 ? (int)(n - i) : 0;
        const Pack<P, 4> pp = load_part<P, 4>(p + i, have, (P)0.f);
        const Pack<G, 4> gg = load_part<G, 4>(g + i, have, (G)0.f);
        Pack<float, 4> m, v;
        int me = 0, ve = 0;
        if (BITS == 8) {
            const int64_t block = first / D1_ADAMW_BLOCK;
            const Pack<uint8_t, 4> mc = load_part<uint8_t, 4>((const uint8_t *)t.m[k] + i, have, 0);
            const Pack<uint8_t, 4> vc = load_part<uint8_t, 4>((const uint8_t *)t.v[k] + i, have, 0);
            me = t.m_exp[k][block];
            ve = t.v_exp[k][block];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                m.v[j] = decode_m(mc.v[j], me);
                v.v[j] = decode<31>(vc.v[j], ve);
            }
        } else {
            m = load_part<float, 4>((const float *)t.m[k] + i, have, 0.f);
            v = load_part<float, 4>((const float *)t.v[k] + i, have, 0.f);
        }
        Pack<P, 4> out;
        Pack<__bf16, 4> half;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float d = (float)gg.v[j] * coef;
            m.v[j] = m.v[j] * r.b1 + d * r.omb1;
            v.v[j] = v.v[j] * r.b2 + (d * d) * r.omb2;
            const float q = (float)pp.v[j] * keep - size * (BITS == 8 ? over8 : over32)(m.v[j], v.v[j], inv2, r.eps);
            out.v[j] = (P)q;
            half.v[j] = (__bf16)q;
        }
        put_part<PAST>(p + i, have, out);
        if (copy) put_part<PAST>(copy + i, have, half);
        if (BITS == 8) {
            // the wave's 256 counters share their upper word but where they pass 2^32
            const uint64_t c0 = (uint64_t)t.counter[k] + (uint64_t)first;
            const uint32_t low = (uint32_t)c0, key = draw_key(r.seed, step, (uint32_t)(c0 >> 32));
            const uint32_t next = low > 0xFFFFFF00u ? draw_key(r.seed, step, (uint32_t)(c0 >> 32) + 1) : key;
            uint32_t word[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t c = low + (threadIdx.x & 63) * 4 + j;
                word[j] = mix(c ^ (c < low ? next : key));
            }
            float ma = 0.f, va = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j < have) {
                    ma = fmaxf(ma, fabsf(m.v[j]));
                    va = fmaxf(va, v.v[j]);
                }
            }
            me = block_exp(lanes_max<64>(ma));
            ve = block_exp(lanes_max<64>(va));
            if ((me > ve ? me : ve) == 255) {      // an infinity (or close to it): the maxima again without
                ma = va = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool lost = !(fabsf(m.v[j]) < INFINITY && v.v[j] < INFINITY);
                    m.v[j] = lost ? 0.f : m.v[j];
                    ma = fmaxf(ma, fabsf(m.v[j]));
                    va = fmaxf(va, lost ? 0.f : v.v[j]);
                    v.v[j] = lost ? INFINITY : v.v[j];
                }
                me = block_exp(lanes_max<64>(ma));
                ve = block_exp(lanes_max<64>(va));
            }
            Pack<uint8_t, 4> mc, vc;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                mc.v[j] = (uint8_t)(encode<15>(fabsf(m.v[j]), me, word[j] >> 16) | (m.v[j] < 0.f ? 128u : 0u));
                const uint32_t code = encode<31>(v.v[j], ve, word[j] & 0xFFFF);
                vc.v[j] = (uint8_t)(code == 0 && v.v[j] > 0.f ? 1 : code);
            }
            put_part<PAST>((uint8_t *)t.m[k] + i, have, mc);
            put_part<PAST>((uint8_t *)t.v[k] + i, have, vc);
            if ((threadIdx.x & 63) == 0) {
                t.m_exp[k][first / D1_ADAMW_BLOCK] = (uint8_t)me;
                t.v_exp[k][first / D1_ADAMW_BLOCK] = (uint8_t)ve;
            }
        } else {
            put_part<PAST>((float *)t.m[k] + i, have, m);
            put_part<PAST>((float *)t.v[k] + i, have, v);
        }
    }
}

// Bound by memory: 98 M fp32 elements in 32 bits 531 us in all, 5.2 TB/s; 369 M with bf16 gradients and copies in 8 bits
// 1,150 us, 5.1 TB/s, there nearly as much by its instructions; small models by two or three launches.
template <int BITS, bool PAST>
__global__ __launch_bounds__(256) void k_adamw_step(const Tensors t, const Rates r, const Join join, int32_t *ctl) {
    __shared__ double s[4];
    float coef;
    int step;
    if (join.parts) {
        double sum = 0.0, c;
        for (int i = threadIdx.x; i < join.count; i += 256) sum += join.parts[i];
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
        __syncthreads();
        const double norm = sqrt((s[0] + s[1]) + (s[2] + s[3]));
        const bool go = clip_of(norm, join.max_norm, c);
        step = ctl[BEFORE] + 1;
        if (join.first && blockIdx.x == 0 && threadIdx.x == 0) {
            ctl[NORM] = __float_as_int((float)norm);
            if (go)
                ctl[STEP] = step;
            else
                ctl[SKIPPED]++;
        }
        if (!go) return;
        coef = (float)c;
    } else {
        if (!ctl[GO]) return;
        coef = __int_as_float(ctl[COEF]);
        step = ctl[STEP];
    }
    int within;
    const int k = tensor_of(t, blockIdx.x, within);
    float inv1 = __int_as_float(ctl[INV_BC1]), inv2 = __int_as_float(ctl[INV_BC2]);
    if (t.lag[k]) corrections(r.log_b1, r.log_b2, step > t.lag[k] ? step - t.lag[k] : 1, inv1, inv2);
    switch (t.types[k]) {
    case 0: return step_chunk<float, float, BITS, PAST>(t, k, within, r, coef, inv1, inv2, (uint32_t)step);
    case 1: return step_chunk<__bf16, float, BITS, PAST>(t, k, within, r, coef, inv1, inv2, (uint32_t)step);
    case 2: return step_chunk<float, __bf16, BITS, PAST>(t, k, within, r, coef, inv1, inv2, (uint32_t)step);
    default: return step_chunk<__bf16, __bf16, BITS, PAST>(t, k, within, r, coef, inv1, inv2, (uint32_t)step);
    }
}

// 369 M codes 341 us, 5.4 TB/s.
template <bool PAST>
__global__ __launch_bounds__(256) void k_adamw_read(const uint8_t *__restrict__ code, const uint8_t *__restrict__ exp, int64_t n,
                                                    int is_signed, float *__restrict__ out) {
    constexpr int ALL = CHUNK / 1024;
    for (int64_t begin = (int64_t)blockIdx.x * CHUNK; begin < n; begin += (int64_t)gridDim.x * CHUNK) {
        Pack<uint8_t, 4> c[ALL];
        int e[ALL], have[ALL];
#pragma unroll
        for (int u = 0; u < ALL; u++) {       // all loads before the first store
            const int64_t i = begin + u * 1024 + threadIdx.x * 4;
            have[u] = n - i >= 4 ? 4 : n - i > 0 ? (int)(n - i) : 0;
            c[u] = load_part<uint8_t, 4>(code + i, have[u], 0);
            e[u] = have[u] ? exp[i / D1_ADAMW_BLOCK] : 0;
        }
#pragma unroll
        for (int u = 0; u < ALL; u++) {
            Pack<float, 4> o;
#pragma unroll
            for (int j = 0; j < 4; j++) o.v[j] = is_signed ? decode_m(c[u].v[j], e[u]) : decode<31>(c[u].v[j], e[u]);
            put_part<PAST>(out + begin + u * 1024 + threadIdx.x * 4, have[u], o);
        }
    }
}

// the next launch's tensors, from t[at]; returns the first tensor it does not hold. Tensors of no
// elements are left out; a launch holds fewer than 2^31 chunks.
inline int take(const D1AdamWTensor *t, int count, int chunk, int at, Tensors &l) {
    l.count = 0;
    l.chunk = chunk;
    int64_t chunks = 0;
    for (; at < count && l.count < MAX_TENSORS; at++) {
        if (t[at].n == 0) continue;
        const int64_t more = (t[at].n + chunk - 1) / chunk;
        if (chunks + more > (1 << 23)) {          // a grid of 2^31 threads
            if (l.count) break;
            return -1;
        }
        const int k = l.count++;
        chunks += more;
        l.p[k] = t[at].p;
        l.g[k] = t[at].g;
        l.m[k] = t[at].m;
        l.v[k] = t[at].v;
        l.m_exp[k] = t[at].m_exp;
        l.v_exp[k] = t[at].v_exp;
        l.copy[k] = t[at].copy;
        l.n[k] = t[at].n;
        l.counter[k] = t[at].counter;
        l.lr[k] = (float)t[at].lr;
        l.keep[k] = (float)(1.0 - t[at].lr * t[at].weight_decay);
        l.lag[k] = t[at].lag;
        l.last_chunk[k] = (int32_t)chunks;
        l.types[k] = (uint8_t)((t[at].ptype == D1_BF16) | (t[at].gtype == D1_BF16) << 1);
    }
    l.chunks = (int32_t)chunks;
    return at;
}
inline int norm_per(const Tensors &l) { return (l.chunks + NORM_GRID - 1) / NORM_GRID; }
inline int norm_blocks(const Tensors &l) { return l.chunks ? (l.chunks + norm_per(l) - 1) / norm_per(l) : 0; }
// Elements a workgroup takes: CHUNK, or a quarter where that leaves the 256 CUs fewer than four workgroups
// each (the policy's 0.53 M elements: step 9.4 us in 130 workgroups, 7.2 in 521).
inline int64_t elements_of(const D1AdamWTensor *t, int count) {
    int64_t n = 0;
    for (int i = 0; i < count; i++) n += t[i].n;
    return n;
}
inline int chunk_of(const D1AdamWTensor *t, int count) {
    return elements_of(t, count) < (int64_t)1024 * CHUNK ? SMALL_CHUNK : CHUNK;
}
// Whether what a step writes is past what the caches hold (20 M elements in 32 bits: 98 us through them, 86 past them; 369 M
// in 8 bits 1,239 and 1,158).
inline bool past_of(const D1AdamWTensor *t, int count, int bits) {
    return elements_of(t, count) * (4 + bits / 4) > PAST_BYTES;
}

}  // namespace d1o

using namespace d1o;

static bool adamw_args(const D1AdamWTensor *t, int count, const D1AdamW *h) {
    if (count < 0 || (count && !t) || !h || (h->bits != 32 && h->bits != 8)) return false;
    if (!(h->beta1 >= 0 && h->beta1 < 1) || !(h->beta2 >= 0 && h->beta2 < 1) || !(h->eps >= 0) || !(h->max_norm >= 0))
        return false;
    for (int i = 0; i < count; i++) {
        const D1AdamWTensor &a = t[i];
        if (a.n < 0 || a.n > (int64_t)CHUNK << 23 || a.lag < 0 || !(a.lr >= 0) || !(a.weight_decay >= 0) || (a.ptype != D1_FP32 && a.ptype != D1_BF16) ||
            (a.gtype != D1_FP32 && a.gtype != D1_BF16))
            return false;
        if (a.n && (!a.p || !a.g || !a.m || !a.v || (h->bits == 8 && (!a.m_exp || !a.v_exp)))) return false;
    }
    return true;
}

extern "C" int64_t d1_adamw_work_bytes(const D1AdamWTensor *t, int count, const D1AdamW *h) {
    if (!adamw_args(t, count, h)) return D1_E_ARG;
    if (!(h->max_norm > 0)) return 0;
    int64_t parts = 0;
    const int chunk = chunk_of(t, count);
    Tensors l;
    for (int at = 0; at < count;) {
        at = take(t, count, chunk, at, l);
        parts += norm_blocks(l);
    }
    return parts * (int64_t)sizeof(double);
}

extern "C" int d1_adamw_step(const D1AdamWTensor *t, int count, const D1AdamW *h, int32_t *ctl, void *work, int64_t work_bytes,
                             void *stream) {
    const int64_t need = d1_adamw_work_bytes(t, count, h);
    if (need < 0 || !ctl || (need && (!work || work_bytes < need || ((uintptr_t)work & 7)))) return D1_E_ARG;
    hipStream_t s = (hipStream_t)stream;
    const double log_b1 = h->beta1 > 0 ? log(h->beta1) : -INFINITY, log_b2 = h->beta2 > 0 ? log(h->beta2) : -INFINITY;
    const int chunk = chunk_of(t, count);
    Tensors l;
    double *parts = h->max_norm > 0 ? (double *)work : nullptr;
    int nparts = 0, e;
    const bool join = parts && need <= JOIN_PARTS * (int64_t)sizeof(double) && need;
    if (parts)
        for (int at = 0; at < count;) {
            at = take(t, count, chunk, at, l);
            if (!l.count) break;
            k_adamw_norm<<<norm_blocks(l), 256, 0, s>>>(l, norm_per(l), parts + nparts, join && !nparts ? ctl : nullptr, log_b1, log_b2);
            if ((e = (int)hipGetLastError())) return e;
            nparts += norm_blocks(l);
        }
    if (!join) {
        k_adamw_begin<<<1, parts ? 1024 : 64, 0, s>>>(ctl, nparts ? parts : nullptr, nparts, h->max_norm, log_b1, log_b2);
        if ((e = (int)hipGetLastError())) return e;
    }
    Join j{join ? parts : nullptr, nparts, 1, h->max_norm};
    const bool past = past_of(t, count, h->bits);
    const Rates r{(float)h->beta1, (float)(1.0 - h->beta1), (float)h->beta2, (float)(1.0 - h->beta2), (float)h->eps,
                  log_b1, log_b2, h->seed};
    for (int at = 0; at < count;) {
        at = take(t, count, chunk, at, l);
        if (!l.count) break;
        if (h->bits == 8 && past)
            k_adamw_step<8, true><<<l.chunks, 256, 0, s>>>(l, r, j, ctl);
        else if (h->bits == 8)
            k_adamw_step<8, false><<<l.chunks, 256, 0, s>>>(l, r, j, ctl);
        else if (past)
            k_adamw_step<32, true><<<l.chunks, 256, 0, s>>>(l, r, j, ctl);
        else
            k_adamw_step<32, false><<<l.chunks, 256, 0, s>>>(l, r, j, ctl);
        if ((e = (int)hipGetLastError())) return e;
        j.first = 0;
    }
    return 0;
}

extern "C" int d1_adamw_read(const uint8_t *code, const uint8_t *exp, int64_t n, int is_signed, float *out, void *stream) {
    if (n < 0 || (is_signed != 0 && is_signed != 1)) return D1_E_ARG;
    if (n == 0) return 0;
    if (!code || !exp || !out) return D1_E_ARG;
    const int64_t need = (n + CHUNK - 1) / CHUNK;
    const unsigned grid = (unsigned)(need < (1 << 20) ? need : (1 << 20));
    if (n * 4 > PAST_BYTES)
        k_adamw_read<true><<<grid, 256, 0, (hipStream_t)stream>>>(code, exp, n, is_signed, out);
    else
        k_adamw_read<false><<<grid, 256, 0, (hipStream_t)stream>>>(code, exp, n, is_signed, out);
    return (int)hipGetLastError();
}
