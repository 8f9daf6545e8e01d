// d1ops: layer norm over rows, forward and backward, gfx950.
//
// With mu and r = 1/sqrt(var + eps) of a row and xh = (x - mu) r:
//   y = xh w + b;  u = dy w;  dx = r (u - mean(u) - xh mean(u xh));  dw = sum dy xh;  db = sum dy.
// Both passes read each input once: a row stays in the registers of LANES lanes (4 to 64 of a
// wave, or a whole workgroup of 256 or 1024), CH chunks of 16 bytes a lane, so the variance is
// taken about the mean itself and not from a difference of sums. The backward pass keeps the
// columns' dw and db sums in registers over all rows that a workgroup walks, writes them once, and
// k_norm_reduce adds the workgroups' sums in a fixed order (no atomics: the same bits each time).
#include "d1_rows.h"

namespace d1o {

constexpr int threads_of(int lanes) { return lanes <= 64 ? 256 : lanes; }
template <class T>
constexpr int vec_of() { return 16 / (int)sizeof(T); }

// sums of a and b over the LANES lanes of a row; `turn` alternates the scratch halves so that one
// barrier a call is enough (a wave is never more than one call ahead)
template <int LANES>
__device__ __forceinline__ void row_sum2(float &a, float &b, float2 (*scratch)[16], int &turn) {
    a = lanes_sum<(LANES < 64 ? LANES : 64)>(a);
    b = lanes_sum<(LANES < 64 ? LANES : 64)>(b);
    if (LANES > 64) {
        float2 *s = scratch[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < LANES / 64; i++) {
            a += s[i].x;
            b += s[i].y;
        }
    }
}

template <class T, class W, int LANES, int CH>
__global__ __launch_bounds__(threads_of(LANES)) void k_norm_fwd(const T *__restrict__ x, int64_t rows, int width, int64_t stride,
                                                                const W *__restrict__ w, const W *__restrict__ b, float eps,
                                                                T *__restrict__ y, float *__restrict__ mean,
                                                                float *__restrict__ rstd) {
    constexpr int VEC = vec_of<T>(), GROUPS = threads_of(LANES) / LANES;
    __shared__ float2 scratch[2][16];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    int turn = 0;
    float wv[CH][VEC], bv[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int col = (c * LANES + lane) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            wv[c][i] = w && col + i < width ? (float)w[col + i] : 1.f;
            bv[c][i] = b && col + i < width ? (float)b[col + i] : 0.f;
        }
    }
    const float inv = 1.f / (float)width;
    for (int64_t row = (int64_t)blockIdx.x * GROUPS + group; row < rows; row += (int64_t)gridDim.x * GROUPS) {
        Pack<T, VEC> a[CH];
        float sum = 0.f, none = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (c * LANES + lane) * VEC;
            a[c] = load_part<T, VEC>(x + row * stride + col, width - col, (T)0.f);
        }
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) sum += (float)a[c].v[i];
        row_sum2<LANES>(sum, none, scratch, turn);
        const float mu = sum * inv;
        float sq = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = (float)a[c].v[i] - mu;
                if ((c * LANES + lane) * VEC + i < width) sq = __builtin_fmaf(d, d, sq);
            }
        row_sum2<LANES>(sq, none, scratch, turn);
        const float r = 1.f / sqrtf(sq * inv + eps);
        if (lane == 0) {
            mean[row] = mu;
            rstd[row] = r;
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (c * LANES + lane) * VEC;
            Pack<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = (T)__builtin_fmaf(((float)a[c].v[i] - mu) * r, wv[c][i], bv[c][i]);
            store_part<T, VEC>(y + row * width + col, width - col, o);
        }
    }
}

template <class T, class W, int LANES, int CH>
__global__ __launch_bounds__(threads_of(LANES)) void k_norm_bwd(const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ x,
                                                                int64_t rows, int width, int64_t stride, const W *__restrict__ w,
                                                                const float *__restrict__ mean, const float *__restrict__ rstd,
                                                                T *__restrict__ dx, float *__restrict__ parts) {
    constexpr int VEC = vec_of<T>(), THREADS = threads_of(LANES), GROUPS = THREADS / LANES, COLS = LANES * CH * VEC;
    __shared__ float2 scratch[2][16];
    __shared__ float sums[GROUPS > 1 ? GROUPS * COLS : 1];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    int turn = 0;
    float wv[CH][VEC], gw[CH][VEC], gb[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int col = (c * LANES + lane) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            wv[c][i] = w && col + i < width ? (float)w[col + i] : 1.f;
            gw[c][i] = gb[c][i] = 0.f;
        }
    }
    const float inv = 1.f / (float)width;
    for (int64_t row = (int64_t)blockIdx.x * GROUPS + group; row < rows; row += (int64_t)gridDim.x * GROUPS) {
        const float mu = mean[row], r = rstd[row];
        Pack<T, VEC> a[CH], g[CH];
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (c * LANES + lane) * VEC;
            a[c] = load_part<T, VEC>(x + row * stride + col, width - col, (T)0.f);
            g[c] = load_part<T, VEC>(dy + row * dy_stride + col, width - col, (T)0.f);
        }
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = (float)g[c].v[i], h = ((float)a[c].v[i] - mu) * r, u = d * wv[c][i];
                gw[c][i] = __builtin_fmaf(d, h, gw[c][i]);
                gb[c][i] += d;
                c1 += u;
                c2 = __builtin_fmaf(u, h, c2);
            }
        row_sum2<LANES>(c1, c2, scratch, turn);
        c1 *= inv;
        c2 *= inv;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (c * LANES + lane) * VEC;
            Pack<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float h = ((float)a[c].v[i] - mu) * r;
                o.v[i] = (T)(r * (__builtin_fmaf((float)g[c].v[i], wv[c][i], -c1) - h * c2));
            }
            store_part<T, VEC>(dx + row * width + col, width - col, o);
        }
    }
    if (!parts) return;
    float *out = parts + (size_t)blockIdx.x * 2 * width;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (GROUPS == 1) {
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const int col = (c * LANES + lane) * VEC + i;
                    if (col < width) out[k * width + col] = k ? gb[c][i] : gw[c][i];
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int i = 0; i < VEC; i++) sums[group * COLS + (c * LANES + lane) * VEC + i] = k ? gb[c][i] : gw[c][i];
            __syncthreads();
            for (int col = threadIdx.x; col < width; col += THREADS) {
                float s = 0.f;
                for (int j = 0; j < GROUPS; j++) s += sums[j * COLS + col];
                out[k * width + col] = s;
            }
        }
    }
}

// the workgroups' column sums parts[nparts][2][width], added: 32 columns a workgroup, each summed
// by 32 threads that take every 32nd part, then over the threads in order
template <class W>
__global__ __launch_bounds__(1024) void k_norm_reduce(const float *__restrict__ parts, int nparts, int width, W *__restrict__ dw,
                                                      W *__restrict__ db) {
    __shared__ float s[32][33];
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
    W *out = blockIdx.y ? db : dw;
    if (!out) return;
    float sum = 0.f;
    if (col < width)
        for (int p = k; p < nparts; p += 32) sum += parts[((size_t)p * 2 + blockIdx.y) * width + col];
    s[k][c] = sum;
    __syncthreads();
    if (k == 0 && col < width) {
        sum = 0.f;
        for (int j = 0; j < 32; j++) sum += s[j][c];
        out[col] = (W)sum;
    }
}

// Row shape for a width: lanes a row and chunks a lane, the fewest that hold it.
#define D1O_NORM_SHAPES(X) X(4, 1) X(16, 1) X(32, 1) X(64, 1) X(64, 2) X(64, 4) X(256, 2) X(256, 4) X(1024, 2) X(1024, 4)
inline int shape_of(int width, int type, int &lanes) {
    const int vec = type == D1_FP32 ? 4 : 8;
#define X(L, C)                     \
    if (width <= (L) * (C) * vec) { \
        lanes = L;                  \
        return C;                   \
    }
    D1O_NORM_SHAPES(X)
#undef X
    return 0;
}

// Workgroups of a pass: at most 4 for each of the 256 CUs, fewer where rows are few.
inline int grid_of(int64_t rows, int lanes) {
    const int groups = threads_of(lanes) / lanes;
    const int64_t need = (rows + groups - 1) / groups;
    const int64_t most = lanes == 1024 ? 512 : 1024;
    return (int)(need < most ? need : most);
}

template <class T, class W>
int fwd(const void *x, int type, int64_t rows, int width, int64_t stride, const void *w, const void *b, float eps, void *y,
        float *mean, float *rstd, hipStream_t s) {
    int lanes = 0;
    const int ch = shape_of(width, type, lanes);
    const dim3 grid(grid_of(rows, lanes));
#define X(L, C)                                                                                                            \
    if constexpr (L * C * vec_of<T>() <= D1_NORM_MAX_WIDTH)                                                                \
        if (lanes == L && ch == C)                                                                                         \
        k_norm_fwd<T, W, L, C><<<grid, threads_of(L), 0, s>>>((const T *)x, rows, width, stride, (const W *)w, (const W *)b, \
                                                              eps, (T *)y, mean, rstd);
    D1O_NORM_SHAPES(X)
#undef X
    return (int)hipGetLastError();
}

template <class T, class W>
int bwd(const void *dy, int64_t dy_stride, const void *x, int type, int64_t rows, int width, int64_t stride, const void *w,
        const float *mean, const float *rstd, void *dx, void *dw, void *db, float *parts, hipStream_t s) {
    int lanes = 0;
    const int ch = shape_of(width, type, lanes), grid = grid_of(rows, lanes);
    if (rows > 0) {
#define X(L, C)                                                                                                          \
    if constexpr (L * C * vec_of<T>() <= D1_NORM_MAX_WIDTH)                                                              \
        if (lanes == L && ch == C)                                                                                       \
        k_norm_bwd<T, W, L, C><<<grid, threads_of(L), 0, s>>>((const T *)dy, dy_stride, (const T *)x, rows, width, stride, \
                                                              (const W *)w, mean, rstd, (T *)dx, parts);
        D1O_NORM_SHAPES(X)
#undef X
        const int e = (int)hipGetLastError();
        if (e) return e;
    }
    if (parts) {
        k_norm_reduce<W><<<dim3((width + 31) / 32, 2), 1024, 0, s>>>(parts, grid, width, (W *)dw, (W *)db);
        return (int)hipGetLastError();
    }
    return 0;
}

}  // namespace d1o

using namespace d1o;

#define D1O_NORM_TYPES(F, ...)                                                          \
    if (type == D1_FP32) return F<float, float>(__VA_ARGS__);                           \
    if (type == D1_BF16)                                                                \
        return wtype == D1_FP32 ? F<__bf16, float>(__VA_ARGS__) : F<__bf16, __bf16>(__VA_ARGS__); \
    return wtype == D1_FP32 ? F<_Float16, float>(__VA_ARGS__) : F<_Float16, _Float16>(__VA_ARGS__);

static bool norm_args(int type, int wtype, int64_t rows, int width, int64_t stride) {
    return is_type(type) && (wtype == type || wtype == D1_FP32) && rows >= 0 && width >= 1 && width <= D1_NORM_MAX_WIDTH &&
           stride >= 0;
}

extern "C" int d1_norm_fwd(const void *x, int type, int64_t rows, int width, int64_t stride, const void *w, const void *b,
                           int wtype, float eps, void *y, float *mean, float *rstd, void *stream) {
    if (!norm_args(type, wtype, rows, width, stride)) return D1_E_ARG;
    if (rows == 0) return 0;
    if (!x || !y || !mean || !rstd) return D1_E_ARG;
    D1O_NORM_TYPES(fwd, x, type, rows, width, stride, w, b, eps, y, mean, rstd, (hipStream_t)stream)
}

extern "C" int64_t d1_norm_work_bytes(int64_t rows, int width, int type) {
    if (!norm_args(type, type, rows, width, 0)) return D1_E_ARG;
    int lanes = 0;
    shape_of(width, type, lanes);
    return (int64_t)grid_of(rows, lanes) * 2 * width * sizeof(float);
}

extern "C" int d1_norm_bwd(const void *dy, int64_t dy_stride, const void *x, int type, int64_t rows, int width, int64_t stride,
                           const void *w, int wtype, const float *mean, const float *rstd, void *dx, void *dw, void *db,
                           void *work, int64_t work_bytes, void *stream) {
    if (!norm_args(type, wtype, rows, width, stride) || dy_stride < 0) return D1_E_ARG;
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return D1_E_ARG;
    if (rows > 0 && (dw || db) && (!work || work_bytes < d1_norm_work_bytes(rows, width, type))) return D1_E_ARG;
    if (rows == 0 && !dw && !db) return 0;
    // no rows: the sums of nothing; `parts` is not read then but marks that dw or db is wanted
    float *parts = dw || db ? (rows ? (float *)work : (float *)(dw ? dw : db)) : nullptr;
    D1O_NORM_TYPES(bwd, dy, dy_stride, x, type, rows, width, stride, w, mean, rstd, dx, dw, db, parts, (hipStream_t)stream)
}
