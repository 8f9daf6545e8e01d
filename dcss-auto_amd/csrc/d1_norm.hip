// d1ops: layer norm over rows, forward and backward, gfx950.
//
// With mu and r = 1/sqrt(var + eps) of a row and xh = (x - mu) r:
//   y = xh w + b;  u = dy w;  dx = r (u - mean(u) - xh mean(u xh));  dw = sum dy xh;  db = sum dy.
// Both passes read each input once: a row stays in the registers of LANES lanes (4 to 64 of a
// wave, or a workgroup of 128 to 1,024), CH chunks of 16 bytes a lane, so the variance is
// taken about the mean itself and not from a difference of sums. The backward pass keeps the
// columns' dw and db sums in registers over all rows that a workgroup walks, writes them once, and
// k_norm_reduce adds the workgroups' sums in a fixed order (no atomics: the same bits each time). These sums are fp32: a
// lane adds its rows alone (16,384 rows of 8,192 over 512 workgroups: 32) and the reduction some 50 parts, so a column's
// error is that of rows/512 + 50 additions; fp64 would take twice the registers of the widest rows, which have none left.
// Backward times are of k_norm_bwd alone where it says so, else of a whole call with the reduction (7 us at 8,192 columns).
#include "d1_rows.h"

namespace d1o {

constexpr int threads_of(int lanes) { return lanes <= 64 ? 256 : lanes; }
// Backward: several rows a workgroup, so that few workgroups (and sums to add) fill the card.
// 5,778 x 861 bf16 with the reduction: 14.1 us on 512 threads, 19.5 on one row's 128; 65,536 x 1,024 78 and 83. On 1,024
// threads the registers of two workgroups a CU do not hold a row of bf16 (204).
constexpr int bwd_threads(int lanes) { return lanes > 512 ? lanes : 512; }
constexpr int bwd_waves(int ch) { return ch == 1 ? 6 : 1; }
// waves a SIMD that the forward pass is held to: two workgroups of 1,024 lanes on a CU
constexpr int fwd_waves(int lanes, int ch) { return lanes == 1024 && ch <= 2 ? 8 : 1; }
template <class T>
constexpr int vec_of() { return 16 / (int)sizeof(T); }

// sums of a and b over the LANES lanes of a row; `turn` alternates the scratch halves so that one
// barrier a call is enough (a wave is never more than one call ahead)
template <int LANES>
__device__ __forceinline__ void row_sum2(float &a, float &b, float2 (*scratch)[16], int &turn) {
    a = lanes_sum<(LANES < 64 ? LANES : 64)>(a);
    b = lanes_sum<(LANES < 64 ? LANES : 64)>(b);
    if (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        float2 *s = scratch[turn];
        turn ^= 1;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) s[wave] = make_float2(a, b);
        __syncthreads();
        // every lane reads the sums of one of its row's waves: WAVES lanes add them like a row of that many lanes
        const float2 v = s[wave / WAVES * WAVES + threadIdx.x % WAVES];
        a = lanes_sum<WAVES>(v.x);
        b = lanes_sum<WAVES>(v.y);
    }
}

// The CH chunks of a lane from a row of `width` elements, `fill` past its end: the backward pass, which has no registers
// left for the places below (16,384 x 8,192 bf16: a call 161 us, 172 with them)
template <class T, int LANES, int CH, int VEC>
__device__ __forceinline__ void read_row(Pack<T, VEC> (&a)[CH], const T *row, int lane, int width, T fill) {
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int col = (c * LANES + lane) * VEC;
        a[c] = load_part<T, VEC>(row + col, width - col, fill);
    }
}

// Where a lane's chunks lie in the forward pass: whole packs, moved back at the row's end so that none passes it and no
// branch keeps a load waiting (16,384 x 4,095 bf16: 61 us, 66 with branches; 7,554 x 11,823 fp16 85 and 97; 32,768 x
// 2,048 50 either way). The first elements of a moved pack are another lane's, left out of the sums and stored twice
// alike. The first half of several chunks always lies inside, since shorter rows take a smaller shape; only the smallest
// shape has rows below a pack.
template <int LANES, int CH, int VEC>
struct Columns {
    int lane, width, back[CH];   // elements by which chunk c is moved back, VEC where it holds none of its own
    __device__ __forceinline__ Columns(int l, int w) : lane(l), width(w) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int past = col(c) + VEC - width;
            back[c] = inside(c) || past <= 0 || (narrow() && !lane) ? 0 : past < VEC && !narrow() ? past : VEC;
        }
    }
    static constexpr bool inside(int c) { return c < CH / 2; }
    __device__ __forceinline__ bool narrow() const { return LANES == 4 && width < VEC; }
    __device__ __forceinline__ int col(int c) const { return (c * LANES + lane) * VEC; }
    __device__ __forceinline__ int at(int c) const {
        return inside(c) || back[c] == 0 ? col(c) : narrow() ? 0 : width - VEC;
    }
    __device__ __forceinline__ bool own(int c, int i) const {
        return inside(c) || (i >= back[c] && (!narrow() || i < width));
    }
    // elements that are stored with chunk c
    __device__ __forceinline__ int stored(int c) const { return !inside(c) && back[c] == VEC ? 0 : narrow() ? width : VEC; }
    template <class T>
    __device__ __forceinline__ void read(Pack<T, VEC> (&a)[CH], const T *row) const {
#pragma unroll
        for (int c = 0; c < CH; c++)
            a[c] = narrow() ? load_part<T, VEC>(row, stored(c), (T)0.f) : load<T, VEC>(row + at(c));
    }
};

template <int VEC, int CH, class T>
__device__ __forceinline__ void fill_row(Pack<T, VEC> (&a)[CH], T value) {
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
        for (int i = 0; i < VEC; i++) a[c].v[i] = value;
}

// One reading, one writing, two sums a row; weight and bias stay in registers over the rows. Bound by memory: 16,384 x 8,192 bf16
// 103 us at best, 5.2 TB/s (115 in a loop of it alone); 65,536 x 256 12 us, 5.5 TB/s; below about 4 us by the launch.
template <class T, class W, int LANES, int CH, bool PAST>
__global__ __launch_bounds__(threads_of(LANES), fwd_waves(LANES, CH)) void k_norm_fwd(const T *__restrict__ x, int64_t rows, int width, int64_t stride,
                                                                const W *__restrict__ w, const W *__restrict__ b, float eps,
                                                                T *__restrict__ y, float *__restrict__ mean,
                                                                float *__restrict__ rstd) {
    constexpr int VEC = vec_of<T>(), GROUPS = threads_of(LANES) / LANES;
    __shared__ float2 scratch[2][16];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const Columns<LANES, CH, VEC> k(lane, width);
    int turn = 0;
    int64_t row = (int64_t)blockIdx.x * GROUPS + group;
    Pack<W, VEC> wv[CH], bv[CH];
    fill_row<VEC, CH>(wv, (W)1.f);
    fill_row<VEC, CH>(bv, (W)0.f);
    if (w) k.read(wv, w);
    if (b) k.read(bv, b);
    const float inv = 1.f / (float)width;
    for (; row < rows; row += step) {
        Pack<T, VEC> a[CH];
        k.read(a, x + row * stride);
        float sum = 0.f, none = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) sum += k.own(c, i) ? (float)a[c].v[i] : 0.f;
        row_sum2<LANES>(sum, none, scratch, turn);
        const float mu = sum * inv;
        float sq = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = k.own(c, i) ? (float)a[c].v[i] - mu : 0.f;
                sq = __builtin_fmaf(d, d, sq);
            }
        row_sum2<LANES>(sq, none, scratch, turn);
        const float r = 1.f / sqrtf(sq * inv + eps);
        if (lane == 0) {
            mean[row] = mu;
            rstd[row] = r;
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
            Pack<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++)
                o.v[i] = (T)__builtin_fmaf(((float)a[c].v[i] - mu) * r, (float)wv[c].v[i], (float)bv[c].v[i]);
            put_part<PAST>(y + row * width + k.at(c), k.stored(c), o);
        }
    }
}

// One reading of x and dy, one writing of dx, two sums a row and two a column. Bound by memory and, where a lane holds
// little, by the number of rows in flight: 16,384 x 8,192 bf16 150 us alone, 5.4 TB/s; 65,536 x 1,024 78 us with the reduction, 5.2 TB/s;
// 1,000,000 x 32 bf16 35 with it, 5.4 TB/s (on 4 lanes, where bwd_waves' bound spills two or three registers to the stack).
template <class T, class W, int LANES, int CH, bool PAST>
__global__ __launch_bounds__(bwd_threads(LANES), bwd_waves(CH)) void k_norm_bwd(const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ x,
                                                                int64_t rows, int width, int64_t stride, const W *__restrict__ w,
                                                                const float *__restrict__ mean, const float *__restrict__ rstd,
                                                                T *__restrict__ dx, float *__restrict__ parts) {
    constexpr int VEC = vec_of<T>(), THREADS = bwd_threads(LANES), GROUPS = THREADS / LANES, COLS = LANES * CH * VEC;
    __shared__ float2 scratch[2][16];
    __shared__ float sums[GROUPS > 1 ? GROUPS * COLS : 1];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int turn = 0;
    Pack<W, VEC> wv[CH];
    fill_row<VEC, CH>(wv, (W)1.f);
    if (w) read_row<W, LANES, CH, VEC>(wv, w, lane, width, (W)1.f);
    float gw[CH][VEC] = {}, gb[CH][VEC] = {};
    const float inv = 1.f / (float)width;
    // all groups of a workgroup make the same number of rounds (the row sums hold barriers)
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < rows; first += step) {
        const int64_t row = first + group;
        const bool have = row < rows;
        const float mu = have ? mean[row] : 0.f, r = have ? rstd[row] : 0.f;
        Pack<T, VEC> a[CH], g[CH];
        read_row<T, LANES, CH, VEC>(a, x + row * stride, lane, have ? width : 0, (T)0.f);
        read_row<T, LANES, CH, VEC>(g, dy + row * dy_stride, lane, have ? width : 0, (T)0.f);
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = (float)g[c].v[i], h = ((float)a[c].v[i] - mu) * r, u = d * (float)wv[c].v[i];
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
                o.v[i] = (T)(r * (__builtin_fmaf((float)g[c].v[i], (float)wv[c].v[i], -c1) - h * c2));
            }
            put_part<PAST>(dx + row * width + col, have ? width - col : 0, o);
        }
    }
    if (!parts) return;
    float *out = parts + (size_t)blockIdx.x * 2 * width;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (GROUPS == 1) {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const int col = (c * LANES + lane) * VEC;
                Pack<float, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; i++) o.v[i] = k ? gb[c][i] : gw[c][i];
                store_part<float, VEC>(out + k * width + col, width - col, o);
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
    if (col < width) {
        const float *at = parts + (size_t)blockIdx.y * width + col;
        int p = k;
        for (; p + 7 * 32 < nparts; p += 8 * 32) {       // eight loads in flight
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = at[(size_t)(p + j * 32) * 2 * width];
#pragma unroll
            for (int j = 0; j < 8; j++) sum += v[j];
        }
        for (; p < nparts; p += 32) sum += at[(size_t)p * 2 * width];
    }
    s[k][c] = sum;
    __syncthreads();
    if (k == 0 && col < width) {
        sum = 0.f;
        for (int j = 0; j < 32; j++) sum += s[j][c];
        out[col] = (W)sum;
    }
}

// Lanes a row and chunks a lane for a width: the fewest lanes that hold it at one chunk each. Few
// registers a lane and many waves do more for the bandwidth than many chunks a lane: 16,384 rows of
// 8,192 bf16 forward 103 us on 1,024 lanes x 1 chunk, 122 on 512 x 2, 136 at best on 256 x 4 (one
// row ahead in registers); backward 161, 179 and 251. Reading a row ahead costs more
// waves than it hides (112 and 198 us on 1,024 x 1), so no shape does.
#define D1O_NORM_SHAPES(X)                                                                                          \
    X(4, 1) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(128, 1) X(256, 1) X(512, 1) X(1024, 1) X(1024, 2) X(1024, 4)
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

inline int64_t groups_of_rows(int64_t rows, int lanes) {
    const int groups = threads_of(lanes) / lanes;
    return (rows + groups - 1) / groups;
}
// Forward: workgroups walk the rows with a stride of the grid; more of them than fit at once even out
// their ends, up to where reading the weights again costs (65,536 x 256 bf16: 14.8 us at 1,024, 14.3 at 4,096, 14.4
// at 8,192; 65,536 x 1,024: 87, 52.3 and 52.9; 16,384 x 8,192: 102, 105 and 111).
inline int fwd_grid(int64_t rows, int lanes) {
    const int64_t need = groups_of_rows(rows, lanes), most = lanes == 1024 ? 1024 : lanes == 512 || lanes < 64 ? 4096 : 8192;
    return (int)(need < most ? need : most);
}
// Backward: each workgroup writes its columns' sums, which k_norm_reduce reads again, so no more than fit at once:
// two or three of 512 threads a CU (65,536 x 1,024 bf16 81.4 us at 512, 78.0 at 768, 90.9 at 1,024), two where the
// rows are few beside the sums (5,778 x 861 14.1, 14.9 and 17.3), two of 1,024 lanes (16,384 x 8,192 174, 161 and 178 at 256, 512
// and 768), one where a lane holds several chunks (7,554 x 11,823 144 at 256, 156 at 512).
inline int bwd_grid(int64_t rows, int lanes, int ch) {
    const int groups = bwd_threads(lanes) / lanes;
    const int64_t need = (rows + groups - 1) / groups, most = ch > 1 ? 256 : lanes <= 512 && rows >= 16384 ? 768 : 512;
    return (int)(need < most ? need : most);
}

// Whether the result goes past the caches: large ones of rows of several chunks a lane (8,192 x 16,384 bf16 forward 100 us
// through the caches, 97 past them, backward 195 and 169; 6,000 x 16,384 fp32 234 and 234). At one chunk a lane it is as fast or slower
// (65,536 x 512 forward 25.7 and 28.3, backward 42.2 and 41.7).
inline bool past_of(int64_t rows, int width, int ch, size_t size) { return ch > 1 && rows * width * (int64_t)size > PAST_BYTES; }

struct Fwd {
    const void *x;
    int64_t rows, stride;
    int width, type;
    const void *w, *b;
    float eps;
    void *y;
    float *mean, *rstd;
    hipStream_t stream;
};
struct Bwd {
    const void *dy, *x;
    int64_t rows, dy_stride, stride;
    int width, type;
    const void *w;
    const float *mean, *rstd;
    void *dx, *dw, *db;
    float *parts;
    hipStream_t stream;
};

template <class T, class W, int LANES, int CH, bool PAST>
void launch(const Fwd &a, int grid) {
    k_norm_fwd<T, W, LANES, CH, PAST><<<grid, threads_of(LANES), 0, a.stream>>>(
        (const T *)a.x, a.rows, a.width, a.stride, (const W *)a.w, (const W *)a.b, a.eps, (T *)a.y, a.mean, a.rstd);
}
template <class T, class W, int LANES, int CH, bool PAST>
void launch(const Bwd &a, int grid) {
    k_norm_bwd<T, W, LANES, CH, PAST><<<grid, bwd_threads(LANES), 0, a.stream>>>(
        (const T *)a.dy, a.dy_stride, (const T *)a.x, a.rows, a.width, a.stride, (const W *)a.w, a.mean, a.rstd, (T *)a.dx,
        a.parts);
}
// the kernel of the rows' shape
template <class T, class W, class Args>
int dispatch(const Args &a, int lanes, int ch, int grid) {
    const bool past = past_of(a.rows, a.width, ch, sizeof(T));
#define X(L, C)                                                           \
    if constexpr (L * C * vec_of<T>() <= D1_NORM_MAX_WIDTH) {             \
        if (lanes == L && ch == C) {                                      \
            if (past)                                                     \
                launch<T, W, L, C, (C > 1)>(a, grid);                     \
            else                                                          \
                launch<T, W, L, C, false>(a, grid);                       \
        }                                                                 \
    }
    D1O_NORM_SHAPES(X)
#undef X
    return (int)hipGetLastError();
}

template <class T, class W>
int run(const Fwd &a) {
    int lanes = 0;
    const int ch = shape_of(a.width, a.type, lanes);
    return dispatch<T, W>(a, lanes, ch, fwd_grid(a.rows, lanes));
}
template <class T, class W>
int run(const Bwd &a) {
    int lanes = 0;
    const int ch = shape_of(a.width, a.type, lanes), grid = bwd_grid(a.rows, lanes, ch);
    if (a.rows > 0) {
        const int e = dispatch<T, W>(a, lanes, ch, grid);
        if (e) return e;
    }
    if (!a.dw && !a.db) return 0;
    k_norm_reduce<W><<<dim3((a.width + 31) / 32, 2), 1024, 0, a.stream>>>(a.parts, grid, a.width, (W *)a.dw, (W *)a.db);
    return (int)hipGetLastError();
}
template <class Args>
int run_types(const Args &a, int wtype) {
    if (a.type == D1_FP32) return run<float, float>(a);
    if (a.type == D1_BF16) return wtype == D1_FP32 ? run<__bf16, float>(a) : run<__bf16, __bf16>(a);
    return wtype == D1_FP32 ? run<_Float16, float>(a) : run<_Float16, _Float16>(a);
}

}  // namespace d1o

using namespace d1o;

static bool norm_args(int type, int wtype, int64_t rows, int width, int64_t stride) {
    return is_type(type) && (wtype == type || wtype == D1_FP32) && rows >= 0 && width >= 1 && width <= D1_NORM_MAX_WIDTH &&
           stride >= 0;
}

extern "C" int d1_norm_fwd(const void *x, int type, int64_t rows, int width, int64_t stride, const void *w, const void *b,
                           int wtype, float eps, void *y, float *mean, float *rstd, void *stream) {
    if (!norm_args(type, wtype, rows, width, stride)) return D1_E_ARG;
    if (rows == 0) return 0;
    if (!x || !y || !mean || !rstd) return D1_E_ARG;
    return run_types(Fwd{x, rows, stride, width, type, w, b, eps, y, mean, rstd, (hipStream_t)stream}, wtype);
}

extern "C" int64_t d1_norm_work_bytes(int64_t rows, int width, int type) {
    if (!norm_args(type, type, rows, width, 0)) return D1_E_ARG;
    int lanes = 0;
    const int ch = shape_of(width, type, lanes);
    return (int64_t)bwd_grid(rows, lanes, ch) * 2 * width * sizeof(float);
}

extern "C" int d1_norm_bwd(const void *dy, int64_t dy_stride, const void *x, int type, int64_t rows, int width, int64_t stride,
                           const void *w, int wtype, const float *mean, const float *rstd, void *dx, void *dw, void *db,
                           void *work, int64_t work_bytes, void *stream) {
    if (!norm_args(type, wtype, rows, width, stride) || dy_stride < 0) return D1_E_ARG;
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return D1_E_ARG;
    if (rows > 0 && (dw || db) && (!work || work_bytes < d1_norm_work_bytes(rows, width, type))) return D1_E_ARG;
    if (rows == 0 && !dw && !db) return 0;
    float *parts = dw || db ? (float *)work : nullptr;
    return run_types(Bwd{dy, x, rows, dy_stride, stride, width, type, w, mean, rstd, dx, dw, db, parts, (hipStream_t)stream}, wtype);
}
