// d1ops: the clipped policy loss with value, entropy and reference-KL terms, and its gradients, gfx950.
//
// For a token with d = logp - old, r = e^d, advantage A and weight w (0 where the mask leaves it out):
//   policy   -min(r A, clip(r, 1 - low, 1 + high) A): -A r while the clip is not active, a constant past it
//   kl       e^x - x - 1 with x = ref - logp (never negative, its mean over samples of the policy is the KL)
//   value    max((v - R)^2, (v' - R)^2) / 2 with v' = v held within value_clip of the old value
//   drift    e^d - d - 1, the same estimate against the old policy
// Which side of a border a token is on is decided in fp64 from the inputs (d against log(1 + high)), so that it does
// not depend on how an exponential rounds. e^x - x - 1 comes from its series near 0, where the difference would cancel.
//
// The weights need the mask's count alone, so one small pass over the mask (a byte a token) comes first and the losses
// and all gradients then take a single pass over the inputs. Sums over tokens are fp64, in a fixed order without atomics:
// the same inputs give the same bits. Bound by memory: 128 x 65,536 fp32 tokens with every term and all gradients take 91 us
// (377 MB, 4.1 TB/s), 2,048 x 16,411 with a mask and a reference 214 us (975 MB, 4.6 TB/s; a large copy 4.8); small calls by
// their launches (8,192 tokens 9.4 + 2.4 us).
#include "d1_rows.h"

namespace d1o {

enum { LOGP, OLD, ADV, REF, ENT, VAL, RET, OLDV, INPUTS };
enum { ABSENT, FLAT, PER_ROW, STRIDED };
enum { S_POLICY, S_VALUE, S_ENTROPY, S_KL, S_CLIPPED, S_DRIFT, SUMS };
constexpr int LOSS_GRID = 1024, COUNT_GRID = 1024, SINGLE = 2048;

struct Input {
    const void *p;
    int64_t row, step;        // strides in elements
    int32_t mode, type;
};
struct Loss {
    Input in[INPUTS];
    Input mask;
    int64_t rows, length, total;
    int64_t jump_rows, jump_t;           // a thread's next tokens: so many rows and tokens on
    double log_low, log_high, vclip;
    float low, high, kl, vcoef, ecoef;
    int32_t sequence, value_clip, by_row, wide;      // wide: gradients in fp32
    void *dlogp, *dentropy, *dvalues;
};

// four tokens from i = row * length + t (row and t only where a.by_row is set); `have` of them are there
struct Where {
    int64_t i, row, t, length;
    int have;
};
// their elements as they lie in memory; converted once all loads are under way
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <bool ANY, class B>
__device__ __forceinline__ void fetch_each(const Input &in, const Where &w, B *out) {
    if (!ANY && in.mode != PER_ROW) {
#pragma unroll
        for (int j = 0; j < 4; j++) out[j] = ((const B *)in.p)[w.i + (j < w.have ? j : w.have - 1)];
        return;
    }
    int64_t row = w.row, t = w.t;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        out[j] = j < w.have ? ((const B *)in.p)[row * in.row + (ANY ? t * in.step : 0)] : (B)0;
        if (++t == w.length) {
            t = 0;
            row++;
        }
    }
}
template <bool ANY>
__device__ __forceinline__ u32x4 fetch(const Input &in, const Where &w) {
    u32x4 r = {0, 0, 0, 0};
    if (in.mode == FLAT && w.have == 4) {
        if (in.type == D1_FP32) {
            __builtin_memcpy(&r, (const float *)in.p + w.i, 16);
        } else {
            uint32_t h[2];
            __builtin_memcpy(h, (const uint16_t *)in.p + w.i, 8);
            r[0] = h[0];
            r[1] = h[1];
        }
    } else if (in.mode != ABSENT) {
        if (in.type == D1_FP32) {
            uint32_t v[4];
            fetch_each<ANY>(in, w, v);
            r = u32x4{v[0], v[1], v[2], v[3]};
        } else {
            uint16_t v[4];
            fetch_each<ANY>(in, w, v);
            r[0] = v[0] | (uint32_t)v[1] << 16;
            r[1] = v[2] | (uint32_t)v[3] << 16;
        }
    }
    return r;
}
template <bool ANY>
__device__ __forceinline__ uint32_t fetch_mask(const Input &in, const Where &w) {
    if (in.mode == ABSENT) return 0x01010101u;
    uint32_t r = 0;
    if (in.mode == FLAT && w.have == 4) {
        __builtin_memcpy(&r, (const uint8_t *)in.p + w.i, 4);
    } else {
        uint8_t v[4];
        fetch_each<ANY>(in, w, v);
        r = v[0] | v[1] << 8 | v[2] << 16 | (uint32_t)v[3] << 24;
    }
    return r;
}
struct Four {
    float v[4];
};
__device__ __forceinline__ Four values_of(u32x4 r, int type) {
    Four f;
    if (type == D1_FP32) {
#pragma unroll
        for (int j = 0; j < 4; j++) f.v[j] = __uint_as_float(r[j]);
    } else if (type == D1_BF16) {
#pragma unroll
        for (int j = 0; j < 4; j++) f.v[j] = __uint_as_float(j & 1 ? r[j >> 1] & 0xFFFF0000u : r[j >> 1] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) f.v[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r[j >> 1] >> (16 * (j & 1))));
    }
    return f;
}
__device__ __forceinline__ void put(void *p, int type, const Where &w, const float *v) {
    if (type == D1_FP32)
        store_part((float *)p + w.i, w.have, Pack<float, 4>{{v[0], v[1], v[2], v[3]}});
    else if (type == D1_BF16)
        store_part((__bf16 *)p + w.i, w.have, Pack<__bf16, 4>{{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]}});
    else
        store_part((_Float16 *)p + w.i, w.have, Pack<_Float16, 4>{{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]}});
}

// e^x: 2^p of the rounded product p = x log2 e times what the rounding dropped, within 2 halves of a step. (Infinities and NaN
// pass through p. The bounds on the rest are for an x whose product passes fp32's range: it is NaN for an infinite one, infinite past
// 2.36e38 either way.) The library's takes half as many instructions again.
__device__ __forceinline__ float exp_of(float x) {
    const float p = x * 1.44269504f, rest = __builtin_fmaf(x, 1.92596299e-8f, __builtin_fmaf(x, 1.44269504f, -p));
    return __builtin_amdgcn_exp2f(p) * __builtin_fmaf(fminf(fmaxf(rest, -1.f), 1.f), 0.693147181f, 1.f);
}
// e^x - x - 1 given e = e^x; `rise` becomes e^x - 1. Below 1/2 the Taylor series to x^9, whose next term is 1e-9 of the
// sum there.
__device__ __forceinline__ float excess(float x, float e, float &rise) {
    float s = 1.f / 362880.f;
    s = __builtin_fmaf(s, x, 1.f / 40320.f);
    s = __builtin_fmaf(s, x, 1.f / 5040.f);
    s = __builtin_fmaf(s, x, 1.f / 720.f);
    s = __builtin_fmaf(s, x, 1.f / 120.f);
    s = __builtin_fmaf(s, x, 1.f / 24.f);
    s = __builtin_fmaf(s, x, 1.f / 6.f);
    s = __builtin_fmaf(s, x, 0.5f);
    const bool near = fabsf(x) < 0.5f;
    s *= x * x;
    rise = near ? s + x : e - 1.f;
    return near ? s : (e - 1.f) - x;
}

template <int THREADS, class T>
__device__ __forceinline__ T block_sum(T x, T *s) {
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    if (THREADS == 64) return x;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    T sum = 0;
#pragma unroll 4
    for (int w = 0; w < THREADS / 64; w++) sum += s[w];
    return sum;
}
// All sums at once: 32 threads each, which add what the workgroup's threads left in LDS (one after another through lane
// moves they took 10 us of a workgroup's end). The result is in thread 32 k's `sum` for k < SUMS.
template <int THREADS>
__device__ __forceinline__ double block_sums(const double *sums, double (*s)[THREADS + 1]) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SUMS; k++) s[k][threadIdx.x] = sums[k];
    __syncthreads();
    double x = 0.0;
    if (threadIdx.x < 32 * SUMS)
#pragma unroll 8
        for (int i = threadIdx.x & 31; i < THREADS; i += 32) x += s[threadIdx.x >> 5][i];
    for (int d = 16; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

__device__ __forceinline__ int bytes_set(uint32_t m) { return __popc((((m & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | m) & 0x80808080u); }

// The mask's counts. Token level: parts[block] = tokens of the block's share. Sequence level: inverse[row] = 1 / tokens (0
// where there is none), and parts[block] = rows with a token among the block's rows (LANES threads a row).
template <int LANES>
__global__ __launch_bounds__(256) void k_loss_count_rows(const Loss a, int64_t *__restrict__ parts, float *__restrict__ inverse) {
    constexpr int ROWS = 256 / LANES;
    __shared__ int64_t s[4];
    const int lane = threadIdx.x % LANES;
    int64_t some = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
        const uint8_t *m = (const uint8_t *)a.mask.p + row * a.mask.row;
        int64_t n = 0;
        if (a.mask.step == 1) {
            int64_t t = (int64_t)lane * 16;
#pragma unroll 4
            for (; t + 16 <= a.length; t += LANES * 16) {
                const Pack<uint32_t, 4> v = load<uint32_t, 4>((const uint32_t *)(m + t));
                n += bytes_set(v.v[0]) + bytes_set(v.v[1]) + bytes_set(v.v[2]) + bytes_set(v.v[3]);
            }
            for (int j = 0; j < 16; j++) n += t + j < a.length && m[t + j];
        } else {
            for (int64_t t = lane; t < a.length; t += LANES) n += m[t * a.mask.step] != 0;
        }
        n = block_sum<LANES>(n, s);
        if (lane == 0) {
            inverse[row] = n ? 1.f / (float)n : 0.f;
            some += n > 0;
        }
    }
    some = block_sum<256>(some, s);
    if (threadIdx.x == 0) parts[blockIdx.x] = some;
}
__global__ __launch_bounds__(256) void k_loss_count(const Loss a, int64_t *__restrict__ parts) {
    __shared__ int64_t s[4];
    int64_t sum = 0;
    if (a.mask.mode == FLAT) {
        const uint8_t *m = (const uint8_t *)a.mask.p;
        int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
#pragma unroll 4
        for (; i + 16 <= a.total; i += (int64_t)gridDim.x * 4096) {
            const Pack<uint32_t, 4> v = load<uint32_t, 4>((const uint32_t *)(m + i));
            sum += bytes_set(v.v[0]) + bytes_set(v.v[1]) + bytes_set(v.v[2]) + bytes_set(v.v[3]);
        }
        for (int j = 0; j < 16; j++) sum += i + j < a.total && m[i + j];
    } else {
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.total; i += (int64_t)gridDim.x * 256)
            sum += ((const uint8_t *)a.mask.p)[i / a.length * a.mask.row + i % a.length * a.mask.step] != 0;
    }
    sum = block_sum<256>(sum, s);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

template <bool VALUES, bool ANY>
__device__ __forceinline__ void four(const Loss &a, const Where &w, float unit, const float *inverse, double *sums) {
    const uint32_t mask = fetch_mask<ANY>(a.mask, w);
    u32x4 raw[INPUTS];
#pragma unroll
    for (int k = 0; k < (VALUES ? INPUTS : VAL); k++) raw[k] = fetch<ANY>(a.in[k], w);
    float weight[4];
#pragma unroll
    for (int j = 0; j < 4; j++) weight[j] = unit;
    if (inverse) {
        int64_t row = w.row, t = w.t;
        float one = inverse[row] * unit;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            weight[j] = one;
            if (++t == w.length && j + 1 < w.have) {
                t = 0;
                one = inverse[++row] * unit;
            }
        }
    }
    Four x[INPUTS];
#pragma unroll
    for (int k = 0; k < (VALUES ? INPUTS : VAL); k++) x[k] = values_of(raw[k], a.in[k].type);
    float dl[4], de[4], dv[4], sum[SUMS] = {};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const bool in = j < w.have && (mask >> (8 * j) & 0xFFu);
        const float wt = in ? weight[j] : 0.f;
        const float logp = x[LOGP].v[j], adv = x[ADV].v[j];
        const double d = (double)logp - (double)x[OLD].v[j];
        const bool past = adv > 0.f ? d > a.log_high : adv < 0.f && d < a.log_low;
        const float df = logp - x[OLD].v[j], r = exp_of(df);
        float g = past ? 0.f : -adv * r, rise;
        const float gain = (past ? (adv > 0.f ? 1.f + a.high : 1.f - a.low) : r) * adv, drift = excess(df, r, rise);
        sum[S_POLICY] -= in ? gain * wt : 0.f;
        sum[S_CLIPPED] += past ? wt : 0.f;
        sum[S_DRIFT] += in ? drift * wt : 0.f;
        if (a.in[REF].mode) {
            const float gap = x[REF].v[j] - logp;
            const float q = excess(gap, exp_of(gap), rise);
            sum[S_KL] += in ? q * wt : 0.f;
            g -= a.kl * rise;
        }
        dl[j] = in ? g * wt : 0.f;
        if (a.in[ENT].mode) {
            sum[S_ENTROPY] += in ? x[ENT].v[j] * wt : 0.f;
            de[j] = -a.ecoef * wt;
        }
        if (VALUES) {
            const double v = x[VAL].v[j], ret = x[RET].v[j];
            double far = v - ret;
            bool free = true;
            if (a.value_clip) {
                const double old = x[OLDV].v[j], gap = v - old;
                if (!(fabs(gap) <= a.vclip) && gap == gap) {
                    const double held = old + (gap > 0.0 ? a.vclip : -a.vclip) - ret;
                    free = !(held * held > far * far);
                    if (!free) far = held;
                }
            }
            const float f = (float)far;
            sum[S_VALUE] += in ? 0.5f * f * f * wt : 0.f;
            dv[j] = in && free ? f * wt * a.vcoef : 0.f;
        }
    }
#pragma unroll
    for (int k = 0; k < SUMS; k++) sums[k] += (double)sum[k];
    if (a.dlogp) put(a.dlogp, a.wide ? D1_FP32 : a.in[LOGP].type, w, dl);
    if (a.dentropy) put(a.dentropy, a.wide ? D1_FP32 : a.in[ENT].type, w, de);
    if (VALUES && a.dvalues) put(a.dvalues, a.wide ? D1_FP32 : a.in[VAL].type, w, dv);
}

// loss, policy, value, entropy, kl, clipped, drift and the count (tokens, or sequences with a token): thread 32 k has sum k
__device__ __forceinline__ void finish(const Loss &a, double sum, double count, float *terms, double *all) {
    if ((threadIdx.x & 31) == 0 && threadIdx.x < 32 * SUMS) {
        all[threadIdx.x >> 5] = sum;
        terms[1 + (threadIdx.x >> 5)] = (float)sum;
    }
    __syncthreads();
    if (threadIdx.x) return;
    terms[0] = (float)(all[S_POLICY] + (double)a.vcoef * all[S_VALUE] - (double)a.ecoef * all[S_ENTROPY] + (double)a.kl * all[S_KL]);
    terms[7] = (float)count;
}

// A single workgroup counts its mask by itself (THREADS 1,024).
template <int THREADS, bool VALUES, bool ANY>
__global__ __launch_bounds__(THREADS) void k_loss(const Loss a, const int64_t *__restrict__ count_parts, int nparts,
                                                  const float *__restrict__ inverse, double *__restrict__ parts, float *__restrict__ terms) {
    __shared__ int64_t si[THREADS / 64];
    __shared__ double sd[SUMS][THREADS + 1], all[SUMS];
    Where w = {((int64_t)blockIdx.x * THREADS + threadIdx.x) * 4, 0, 0, a.length, 4};
    if (a.by_row) {
        w.row = w.i / a.length;
        w.t = w.i - w.row * a.length;
    }
    int64_t count = a.sequence && a.length ? a.rows : a.total;
    if (nparts) {
        count = 0;
        for (int i = threadIdx.x; i < nparts; i += THREADS) count += count_parts[i];
        count = block_sum<THREADS>(count, si);
    } else if (THREADS == 1024 && a.mask.mode) {
        count = 0;
        for (Where v = w; v.i < a.total; v.i += THREADS * 4) {
            v.have = a.total - v.i < 4 ? (int)(a.total - v.i) : 4;
            uint32_t m = fetch_mask<ANY>(a.mask, v);
            if (v.have < 4) m &= (1u << (8 * v.have)) - 1;
            count += bytes_set(m);
            v.row += a.jump_rows;
            v.t += a.jump_t;
            if (v.t >= a.length) {
                v.t -= a.length;
                v.row++;
            }
        }
        count = block_sum<THREADS>(count, si);
    }
    // every sequence alike without a mask: 1 / (length x rows)
    const float unit = (float)(1.0 / (a.sequence && !inverse && !a.mask.mode ? (double)a.total : count > 0 ? (double)count : 1.0));
    double sums[SUMS] = {};
    for (; w.i < a.total; w.i += (int64_t)gridDim.x * THREADS * 4) {
        w.have = a.total - w.i < 4 ? (int)(a.total - w.i) : 4;
        four<VALUES, ANY>(a, w, unit, inverse, sums);
        w.row += a.jump_rows;
        w.t += a.jump_t;
        if (w.t >= a.length) {
            w.t -= a.length;
            w.row++;
        }
    }
    const double sum = block_sums<THREADS>(sums, sd);
    if (a.sequence && a.rows == 1) count = count > 0;
    if (gridDim.x == 1) return finish(a, sum, (double)count, terms, all);
    if ((threadIdx.x & 31) == 0 && threadIdx.x < 32 * SUMS) parts[(int64_t)(threadIdx.x >> 5) * gridDim.x + blockIdx.x] = sum;
    if (blockIdx.x == 0 && threadIdx.x == 0) parts[(int64_t)SUMS * gridDim.x] = (double)count;
}

__global__ __launch_bounds__(256) void k_loss_finish(const Loss a, const double *__restrict__ parts, int n, float *__restrict__ terms) {
    __shared__ double sd[SUMS][257], all[SUMS];
    double sums[SUMS];
#pragma unroll
    for (int k = 0; k < SUMS; k++) {
        double x[LOSS_GRID / 256];
#pragma unroll
        for (int u = 0; u < LOSS_GRID / 256; u++) {
            const int i = u * 256 + threadIdx.x;
            x[u] = i < n ? parts[(int64_t)k * n + i] : 0.0;
        }
        sums[k] = 0.0;
#pragma unroll
        for (int u = 0; u < LOSS_GRID / 256; u++) sums[k] += x[u];
    }
    const double sum = block_sums<256>(sums, sd);
    finish(a, sum, parts[(int64_t)SUMS * n], terms, all);
}

// Gradients made for a loss gradient of 1, scaled by the real one. They are kept in fp32 until then (`type` then is D1_FP32) and rounded
// to their own type here: a weight of 1 / tokens leaves fp16 few bits, or none, which a factor behind the rounding does not bring back (at
// 2^20 tokens, scaled by 65,536, 1.8% off; 0.02% so). It reads and writes every gradient once more: 128 x 65,536 fp32 tokens with
// every term take 138 us forward and backward through autograd, 99 in the one pass that gives the gradients themselves.
__global__ __launch_bounds__(256) void k_loss_scale(const void *p, int type, void *out, int out_type, int64_t n, const float *__restrict__ by) {
    const float f = *by;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
        const Where w = {i, 0, 0, n, n - i < 4 ? (int)(n - i) : 4};
        const u32x4 r = fetch<false>({p, 0, 1, FLAT, type}, w);
        Four x = values_of(r, type);
#pragma unroll
        for (int j = 0; j < 4; j++) x.v[j] *= f;
        put(out, out_type, w, x.v);
    }
}

inline int loss_grid(int64_t total) {
    const int64_t n = (total + 1023) / 1024;
    return (int)(n < LOSS_GRID ? n : LOSS_GRID);
}
// A sequence alone is its tokens. Rows are counted by a wave each, long ones by a workgroup.
inline bool rows_counted(const D1PolicyLoss *h) { return h->sequence && h->rows > 1 && h->mask.data; }
inline bool rows_long(const D1PolicyLoss *h) { return h->length > 8192; }
inline int count_grid(const D1PolicyLoss *h) {
    const int64_t n = !rows_counted(h) ? (h->rows * h->length + 16383) / 16384 : rows_long(h) ? h->rows : (h->rows + 3) / 4;
    return (int)(n < 1 ? 1 : n < COUNT_GRID ? n : COUNT_GRID);
}
// One workgroup of 1,024 threads does all in one launch, but for the counts of several sequences (8,192 tokens with every term
// would take it 17 us, 8 workgroups and the join 9).
inline bool is_single(const D1PolicyLoss *h) {
    const int64_t total = h->rows * h->length;
    return total == 0 || (total <= SINGLE && !rows_counted(h));
}

static bool loss_args(const D1PolicyLoss *h) {
    if (!h || h->rows < 0 || h->length < 0 || (h->sequence != 0 && h->sequence != 1) || (h->fp32_grads != 0 && h->fp32_grads != 1)) return false;
    if (h->length && h->rows > ((int64_t)1 << 48) / h->length) return false;
    if (!(h->clip_low >= 0 && h->clip_low <= 1 && h->clip_high >= 0) || !(h->value_clip >= 0)) return false;
    for (double c : {h->kl_coef, h->value_coef, h->entropy_coef})
        if (!(c - c == 0)) return false;
    const bool some = h->rows && h->length;
    if (some && (!h->logp.data || !h->old_logp.data || !h->advantages.data)) return false;
    if (some && (!h->values.data != !h->returns.data || (h->value_clip > 0 && h->values.data && !h->old_values.data))) return false;
    for (const D1LossInput *t : {&h->logp, &h->old_logp, &h->advantages, &h->ref_logp, &h->entropy, &h->values, &h->returns, &h->old_values})
        if (t->data && (!is_type(t->type) || t->row < 0 || t->step < 0)) return false;
    return !h->mask.data || (h->mask.row >= 0 && h->mask.step >= 0);
}

static Input input(const D1LossInput &t, const D1PolicyLoss *h) {
    Input in{t.data, t.row, t.step, ABSENT, t.type};
    if (t.data)
        in.mode = (t.step == 1 || h->length <= 1) && (t.row == h->length || h->rows <= 1) ? FLAT : t.step == 0 ? PER_ROW : STRIDED;
    return in;
}

template <int THREADS>
static void loss_launch(const Loss &a, bool any, int grid, const int64_t *count_parts, int nparts, const float *inverse, double *parts,
                        float *terms, hipStream_t stream) {
    const dim3 g(grid), b(THREADS);
    if (a.in[VAL].mode && any)
        hipLaunchKernelGGL((k_loss<THREADS, true, true>), g, b, 0, stream, a, count_parts, nparts, inverse, parts, terms);
    else if (a.in[VAL].mode)
        hipLaunchKernelGGL((k_loss<THREADS, true, false>), g, b, 0, stream, a, count_parts, nparts, inverse, parts, terms);
    else if (any)
        hipLaunchKernelGGL((k_loss<THREADS, false, true>), g, b, 0, stream, a, count_parts, nparts, inverse, parts, terms);
    else
        hipLaunchKernelGGL((k_loss<THREADS, false, false>), g, b, 0, stream, a, count_parts, nparts, inverse, parts, terms);
}

}  // namespace d1o

using namespace d1o;

extern "C" {
int64_t d1_policy_loss_work_bytes(const D1PolicyLoss *h) {
    if (!loss_args(h)) return D1_E_ARG;
    const int64_t total = h->rows * h->length;
    if (is_single(h)) return 0;
    return (int64_t)sizeof(double) * (SUMS * loss_grid(total) + 1) +
           (h->mask.data ? (int64_t)sizeof(int64_t) * count_grid(h) + (rows_counted(h) ? (int64_t)sizeof(float) * h->rows : 0) : 0);
}

int d1_policy_loss(const D1PolicyLoss *h, float *terms, void *dlogp, void *dentropy, void *dvalues, void *work, int64_t work_bytes,
                   void *stream_) {
    if (!loss_args(h) || !terms || ((uintptr_t)terms & 3)) return D1_E_ARG;
    if ((dentropy && !h->entropy.data) || (dvalues && !h->values.data)) {
        if (h->rows && h->length) return D1_E_ARG;
    }
    const int64_t need = d1_policy_loss_work_bytes(h);
    if (need > 0 && (!work || work_bytes < need || ((uintptr_t)work & 7))) return D1_E_ARG;
    hipStream_t stream = (hipStream_t)stream_;
    Loss a{};
    const D1LossInput *in[INPUTS] = {&h->logp, &h->old_logp, &h->advantages, &h->ref_logp, &h->entropy, &h->values, &h->returns, &h->old_values};
    for (int k = 0; k < INPUTS; k++) a.in[k] = input(*in[k], h);
    a.mask = input(h->mask, h);
    a.rows = h->rows;
    a.length = h->length;
    a.total = h->rows * h->length;
    a.log_low = log1p(-h->clip_low);
    a.log_high = log1p(h->clip_high);
    a.low = (float)h->clip_low;
    a.high = (float)h->clip_high;
    a.value_clip = h->value_clip > 0;
    a.vclip = h->value_clip;
    a.kl = (float)h->kl_coef;
    a.vcoef = (float)h->value_coef;
    a.ecoef = (float)h->entropy_coef;
    a.sequence = h->sequence;
    a.wide = h->fp32_grads;
    a.dlogp = dlogp;
    a.dentropy = dentropy;
    a.dvalues = dvalues;
    bool any = a.mask.mode == STRIDED || a.mask.mode == PER_ROW, rows = any;
    for (const Input &in : a.in) {
        any |= in.mode == STRIDED;
        rows |= in.mode == STRIDED || in.mode == PER_ROW;
    }
    const bool single = is_single(h);
    const int grid = single ? 1 : loss_grid(a.total), nparts = !single && a.mask.mode ? count_grid(h) : 0;
    double *parts = (double *)work;
    int64_t *count_parts = (int64_t *)(parts + SUMS * grid + 1);
    float *inverse = nparts && rows_counted(h) ? (float *)(count_parts + nparts) : nullptr;
    a.by_row = rows || inverse;
    if (a.by_row) {
        const int64_t jump = (int64_t)grid * (single ? 1024 : 256) * 4;
        a.jump_rows = a.length ? jump / a.length : 0;
        a.jump_t = a.length ? jump % a.length : 0;
    }
    if (inverse && rows_long(h))
        hipLaunchKernelGGL(k_loss_count_rows<256>, dim3(nparts), dim3(256), 0, stream, a, count_parts, inverse);
    else if (inverse)
        hipLaunchKernelGGL(k_loss_count_rows<64>, dim3(nparts), dim3(256), 0, stream, a, count_parts, inverse);
    else if (nparts)
        hipLaunchKernelGGL(k_loss_count, dim3(nparts), dim3(256), 0, stream, a, count_parts);
    if (single)
        loss_launch<1024>(a, any, 1, nullptr, 0, nullptr, nullptr, terms, stream);
    else
        loss_launch<256>(a, any, grid, count_parts, nparts, inverse, parts, terms, stream);
    if (grid > 1) hipLaunchKernelGGL(k_loss_finish, dim3(1), dim3(256), 0, stream, a, parts, grid, terms);
    return (int)hipGetLastError();
}

static int scale(const void *data, int type, void *out, int out_type, int64_t n, const float *by, void *stream) {
    if (n < 0 || !is_type(type) || !is_type(out_type) || (n && (!data || !out || !by))) return D1_E_ARG;
    if (n == 0) return 0;
    const int64_t groups = (n + 1023) / 1024;
    hipLaunchKernelGGL(k_loss_scale, dim3((unsigned)(groups < 2048 ? groups : 2048)), dim3(256), 0, (hipStream_t)stream, data, type, out,
                       out_type, n, by);
    return (int)hipGetLastError();
}
int d1_scale(const void *data, void *out, int type, int64_t n, const float *by, void *stream) {
    return scale(data, type, out, type, n, by, stream);
}
int d1_scale_to(const float *data, void *out, int type, int64_t n, const float *by, void *stream) {
    return scale(data, D1_FP32, out, type, n, by, stream);
}
}
