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
// the same inputs give the same bits. Bound by memory.
#include "d1_rows.h"

namespace d1o {

enum { LOGP, OLD, ADV, REF, ENT, VAL, RET, OLDV, INPUTS };
enum { ABSENT, FLAT, PER_ROW, STRIDED };
enum { S_POLICY, S_VALUE, S_ENTROPY, S_KL, S_CLIPPED, S_DRIFT, SUMS };
constexpr int LOSS_GRID = 1024, COUNT_GRID = 1024, SINGLE = 4096;

struct Input {
    const void *p;
    int64_t row, step;        // strides in elements
    int32_t mode, type;
};
struct Loss {
    Input in[INPUTS];
    Input mask;
    int64_t rows, length, total;
    double log_low, log_high, vclip, inv_length;
    float low, high, kl, vcoef, ecoef;
    int32_t sequence, value_clip;
    void *dlogp, *dentropy, *dvalues;
};

// i = row * length + t for i < 2^52
__device__ __forceinline__ int64_t row_of(int64_t i, int64_t length, double inv_length, int64_t &t) {
    int64_t row = (int64_t)((double)i * inv_length);
    t = i - row * length;
    if (t < 0) {
        row--;
        t += length;
    } else if (t >= length) {
        row++;
        t -= length;
    }
    return row;
}

// four tokens' elements as they lie in memory; converted once all loads are under way
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct Where {
    int64_t i, row, t, length;
    int have;                 // of the four
};
template <class B>
__device__ __forceinline__ void fetch_strided(const Input &in, const Where &w, B *out) {
    int64_t row = w.row, t = w.t;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        out[j] = j < w.have ? ((const B *)in.p)[row * in.row + t * in.step] : (B)0;
        if (++t == w.length) {
            t = 0;
            row++;
        }
    }
}
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
            fetch_strided<uint32_t>(in, w, v);
            r = u32x4{v[0], v[1], v[2], v[3]};
        } else {
            uint16_t v[4];
            fetch_strided<uint16_t>(in, w, v);
            r[0] = v[0] | (uint32_t)v[1] << 16;
            r[1] = v[2] | (uint32_t)v[3] << 16;
        }
    }
    return r;
}
__device__ __forceinline__ uint32_t fetch_mask(const Input &in, const Where &w) {
    if (in.mode == ABSENT) return 0x01010101u;
    uint32_t r = 0;
    if (in.mode == FLAT && w.have == 4) {
        __builtin_memcpy(&r, (const uint8_t *)in.p + w.i, 4);
    } else {
        uint8_t v[4];
        fetch_strided<uint8_t>(in, w, v);
        r = v[0] | v[1] << 8 | v[2] << 16 | (uint32_t)v[3] << 24;
    }
    return r;
}
__device__ __forceinline__ float value_of(u32x4 r, int j, int type) {
    if (type == D1_FP32) return __uint_as_float(r[j]);
    const uint32_t h = r[j >> 1] >> (16 * (j & 1)) & 0xFFFFu;
    return type == D1_BF16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
__device__ __forceinline__ void put(void *p, int type, const Where &w, const float *v) {
    if (type == D1_FP32) {
        Pack<float, 4> a = {{v[0], v[1], v[2], v[3]}};
        store_part<float, 4>((float *)p + w.i, w.have, a);
    } else if (type == D1_BF16) {
        Pack<__bf16, 4> a = {{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]}};
        store_part<__bf16, 4>((__bf16 *)p + w.i, w.have, a);
    } else {
        Pack<_Float16, 4> a = {{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]}};
        store_part<_Float16, 4>((_Float16 *)p + w.i, w.have, a);
    }
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
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    T sum = 0;
    for (int w = 0; w < THREADS / 64; w++) sum += s[w];
    return sum;
}

__device__ __forceinline__ int bytes_set(uint32_t m) {
    return ((m & 0xFFu) != 0) + ((m & 0xFF00u) != 0) + ((m & 0xFF0000u) != 0) + ((m & 0xFF000000u) != 0);
}

// The mask's counts. Token level: parts[block] = tokens of the block's share. Sequence level: counts[row], and
// parts[block] = rows with a token among the block's rows (a wave a row).
__global__ __launch_bounds__(256) void k_loss_count(const Loss a, int64_t *__restrict__ parts, int64_t *__restrict__ counts) {
    __shared__ int64_t s[4];
    int64_t sum = 0;
    if (a.sequence) {
        for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.rows; row += (int64_t)gridDim.x * 4) {
            int64_t n = 0;
            for (int64_t t = (threadIdx.x & 63) * 4; t < a.length; t += 256) {
                const int have = a.length - t < 4 ? (int)(a.length - t) : 4;
                n += bytes_set(fetch_mask(a.mask, {row * a.length + t, row, t, a.length, have}));
            }
            for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
            if ((threadIdx.x & 63) == 0) {
                counts[row] = n;
                sum += n > 0;
            }
        }
    } else {
        for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < a.total; i += (int64_t)gridDim.x * 1024) {
            Where w = {i, 0, 0, a.length, a.total - i < 4 ? (int)(a.total - i) : 4};
            if (a.mask.mode != FLAT || w.have < 4) w.row = row_of(i, a.length, a.inv_length, w.t);
            sum += bytes_set(fetch_mask(a.mask, w));
        }
    }
    sum = block_sum<256>(sum, s);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

template <bool GRAD>
__device__ __forceinline__ void four(const Loss &a, const Where &w, float unit, const int64_t *counts, double rows_some, double *sums) {
    const uint32_t mask = fetch_mask(a.mask, w);
    u32x4 raw[INPUTS];
#pragma unroll
    for (int k = 0; k < INPUTS; k++) raw[k] = fetch(a.in[k], w);
    float weight[4];
    if (counts) {
        int64_t row = w.row, t = w.t;
        float one = 0.f;
        for (int j = 0; j < 4; j++) {
            if (j == 0 || t == 0) one = j < w.have ? (float)(1.0 / ((double)counts[row] * rows_some)) : 0.f;
            weight[j] = one;
            if (++t == w.length) {
                t = 0;
                row++;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) weight[j] = unit;
    }
    float dl[4], de[4], dv[4], sum[SUMS] = {};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const bool in = j < w.have && (mask >> (8 * j) & 0xFFu);
        const float wt = in ? weight[j] : 0.f;
        const float logp = value_of(raw[LOGP], j, a.in[LOGP].type), adv = value_of(raw[ADV], j, a.in[ADV].type);
        const double d = (double)logp - (double)value_of(raw[OLD], j, a.in[OLD].type);
        const bool past = adv > 0.f ? d > a.log_high : adv < 0.f && d < a.log_low;
        const float df = (float)d, r = expf(df);
        float g = past ? 0.f : -adv * r;
        if (in) {
            sum[S_POLICY] -= (past ? (adv > 0.f ? 1.f + a.high : 1.f - a.low) : r) * adv * wt;
            sum[S_CLIPPED] += past ? wt : 0.f;
            float rise;
            sum[S_DRIFT] += excess(df, r, rise) * wt;
        }
        if (a.in[REF].mode) {
            const float x = (float)((double)value_of(raw[REF], j, a.in[REF].type) - (double)logp);
            float rise;
            const float q = excess(x, expf(x), rise);
            if (in) sum[S_KL] += q * wt;
            g -= a.kl * rise;
        }
        dl[j] = in ? g * wt : 0.f;
        if (a.in[ENT].mode) {
            if (in) sum[S_ENTROPY] += value_of(raw[ENT], j, a.in[ENT].type) * wt;
            de[j] = -a.ecoef * wt;
        }
        if (a.in[VAL].mode) {
            const double v = value_of(raw[VAL], j, a.in[VAL].type), ret = value_of(raw[RET], j, a.in[RET].type);
            double far = v - ret;
            bool free = true;
            if (a.value_clip) {
                const double old = value_of(raw[OLDV], j, a.in[OLDV].type), gap = v - old;
                if (!(fabs(gap) <= a.vclip) && gap == gap) {
                    const double held = old + (gap > 0.0 ? a.vclip : -a.vclip) - ret;
                    free = !(held * held > far * far);
                    if (!free) far = held;
                }
            }
            const float f = (float)far;
            if (in) sum[S_VALUE] += 0.5f * f * f * wt;
            dv[j] = in && free ? f * wt * a.vcoef : 0.f;
        }
    }
#pragma unroll
    for (int k = 0; k < SUMS; k++) sums[k] += (double)sum[k];
    if (GRAD) {
        if (a.dlogp) put(a.dlogp, a.in[LOGP].type, w, dl);
        if (a.dentropy) put(a.dentropy, a.in[ENT].type, w, de);
        if (a.dvalues) put(a.dvalues, a.in[VAL].type, w, dv);
    }
}

// loss, policy, value, entropy, kl, clipped, drift and the count (tokens, or sequences with a token)
__device__ __forceinline__ void finish(const Loss &a, const double *sums, double count, float *terms) {
    terms[0] = (float)(sums[S_POLICY] + (double)a.vcoef * sums[S_VALUE] - (double)a.ecoef * sums[S_ENTROPY] + (double)a.kl * sums[S_KL]);
    for (int k = 0; k < SUMS; k++) terms[1 + k] = (float)sums[k];
    terms[7] = (float)count;
}

template <int THREADS, bool GRAD>
__global__ __launch_bounds__(THREADS) void k_loss(const Loss a, const int64_t *__restrict__ count_parts, int nparts,
                                                  const int64_t *__restrict__ counts, double *__restrict__ parts, float *__restrict__ terms) {
    __shared__ int64_t si[THREADS / 64];
    __shared__ double sd[THREADS / 64];
    int64_t count = a.sequence && a.length ? a.rows : a.total;
    if (nparts) {
        count = 0;
        for (int i = threadIdx.x; i < nparts; i += THREADS) count += count_parts[i];
        count = block_sum<THREADS>(count, si);
    } else if (a.mask.mode && THREADS == 1024) {        // the only workgroup counts by itself
        count = 0;
        for (int64_t i = (int64_t)threadIdx.x * 4; i < a.total; i += THREADS * 4) {
            Where w = {i, 0, 0, a.length, a.total - i < 4 ? (int)(a.total - i) : 4};
            w.row = row_of(i, a.length, a.inv_length, w.t);
            count += bytes_set(fetch_mask(a.mask, w));
        }
        count = block_sum<THREADS>(count, si);
    }
    // every sequence alike without a mask: 1 / (length x rows)
    const float unit = (float)(1.0 / (a.sequence && !counts ? (double)a.total : count > 0 ? (double)count : 1.0));
    double sums[SUMS] = {};
    for (int64_t i = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * 4; i < a.total; i += (int64_t)gridDim.x * THREADS * 4) {
        Where w = {i, 0, 0, a.length, a.total - i < 4 ? (int)(a.total - i) : 4};
        w.row = row_of(i, a.length, a.inv_length, w.t);
        four<GRAD>(a, w, unit, counts, (double)count, sums);
    }
#pragma unroll
    for (int k = 0; k < SUMS; k++) sums[k] = block_sum<THREADS>(sums[k], sd);
    if (threadIdx.x) return;
    if (gridDim.x == 1)
        return finish(a, sums, (double)count, terms);
    for (int k = 0; k < SUMS; k++) parts[(int64_t)k * gridDim.x + blockIdx.x] = sums[k];
    if (blockIdx.x == 0) parts[(int64_t)SUMS * gridDim.x] = (double)count;
}

__global__ __launch_bounds__(1024) void k_loss_finish(const Loss a, const double *__restrict__ parts, int n, float *__restrict__ terms) {
    __shared__ double sd[16];
    double sums[SUMS];
#pragma unroll
    for (int k = 0; k < SUMS; k++) {
        double x = 0.0;
        for (int i = threadIdx.x; i < n; i += 1024) x += parts[(int64_t)k * n + i];
        sums[k] = x;
    }
#pragma unroll
    for (int k = 0; k < SUMS; k++) sums[k] = block_sum<1024>(sums[k], sd);
    if (threadIdx.x == 0) finish(a, sums, parts[(int64_t)SUMS * n], terms);
}

// Gradients made for a loss gradient of 1, scaled by the real one; nothing is read or written where that is 1.
__global__ __launch_bounds__(256) void k_loss_scale(void *p, int type, int64_t n, const float *__restrict__ by) {
    const float f = *by;
    if (f == 1.f) return;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
        const Where w = {i, 0, i, n, n - i < 4 ? (int)(n - i) : 4};
        const u32x4 r = fetch({p, 0, 1, FLAT, type}, w);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = value_of(r, j, type) * f;
        put(p, type, w, v);
    }
}

inline int loss_grid(int64_t total) {
    const int64_t n = (total + 1023) / 1024;
    return (int)(n < LOSS_GRID ? n : LOSS_GRID);
}
inline int count_grid(const D1PolicyLoss *h) {
    const int64_t n = h->sequence ? (h->rows + 3) / 4 : (h->rows * h->length + 4095) / 4096;
    return (int)(n < 1 ? 1 : n < COUNT_GRID ? n : COUNT_GRID);
}
// One workgroup of 1,024 threads does all in one launch. A mask by sequences has counts a row to keep.
inline bool is_single(const D1PolicyLoss *h) {
    const int64_t total = h->rows * h->length;
    return total == 0 || (total <= SINGLE && !(h->sequence && h->mask.data));
}

static bool loss_args(const D1PolicyLoss *h) {
    if (!h || h->rows < 0 || h->length < 0 || (h->sequence != 0 && h->sequence != 1)) return false;
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
        in.mode = (t.step == 1 || h->length <= 1) && (t.row == h->length || h->rows <= 1) ? FLAT : STRIDED;
    return in;
}

}  // namespace d1o

using namespace d1o;

extern "C" {
int64_t d1_policy_loss_work_bytes(const D1PolicyLoss *h) {
    if (!loss_args(h)) return D1_E_ARG;
    const int64_t total = h->rows * h->length;
    if (is_single(h)) return 0;
    return (int64_t)sizeof(double) * (SUMS * loss_grid(total) + 1) +
           (h->mask.data ? (int64_t)sizeof(int64_t) * (count_grid(h) + (h->sequence ? h->rows : 0)) : 0);
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
    a.inv_length = h->length ? 1.0 / (double)h->length : 0.0;
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
    a.dlogp = dlogp;
    a.dentropy = dentropy;
    a.dvalues = dvalues;
    const bool grad = dlogp || dentropy || dvalues;
    if (is_single(h)) {
        if (grad)
            hipLaunchKernelGGL((k_loss<1024, true>), dim3(1), dim3(1024), 0, stream, a, nullptr, 0, nullptr, nullptr, terms);
        else
            hipLaunchKernelGGL((k_loss<1024, false>), dim3(1), dim3(1024), 0, stream, a, nullptr, 0, nullptr, nullptr, terms);
        return (int)hipGetLastError();
    }
    const int grid = loss_grid(a.total), nparts = a.mask.mode ? count_grid(h) : 0;
    double *parts = (double *)work;
    int64_t *count_parts = (int64_t *)(parts + SUMS * grid + 1);
    int64_t *counts = a.mask.mode && a.sequence ? count_parts + nparts : nullptr;
    if (nparts) hipLaunchKernelGGL(k_loss_count, dim3(nparts), dim3(256), 0, stream, a, count_parts, counts);
    if (grad)
        hipLaunchKernelGGL((k_loss<256, true>), dim3(grid), dim3(256), 0, stream, a, count_parts, nparts, counts, parts, terms);
    else
        hipLaunchKernelGGL((k_loss<256, false>), dim3(grid), dim3(256), 0, stream, a, count_parts, nparts, counts, parts, terms);
    if (grid > 1) hipLaunchKernelGGL(k_loss_finish, dim3(1), dim3(1024), 0, stream, a, parts, grid, terms);
    return (int)hipGetLastError();
}

int d1_scale(void *data, int type, int64_t n, const float *by, void *stream) {
    if (n < 0 || !is_type(type) || (n && (!data || !by))) return D1_E_ARG;
    if (n == 0) return 0;
    const int64_t groups = (n + 1023) / 1024;
    hipLaunchKernelGGL(k_loss_scale, dim3((unsigned)(groups < 2048 ? groups : 2048)), dim3(256), 0, (hipStream_t)stream, data, type, n, by);
    return (int)hipGetLastError();
}
}
