// d1ops: updates orthogonalised by Newton-Schulz products, and the momentum step made of them, gfx950.
//
// X = U / (|U|_F + eps), on the side with fewer rows; then `steps` times, with (a, b, c) an odd quintic's coefficients that
// pull every singular value towards 1:
//   A = X X^T;  B = a I + b A + c A A;  X = B X
// Matrix instructions take 16-bit operands. A value is held as fp16 (one term: for results in 16 bits, 11 bits of
// mantissa where bf16 would leave 8), or as the sum of two fp16 halves (for results in 32 bits, and of a short side under 16): hi = fp16(v),
// lo = fp16(v - hi), 22 bits, and a product is hi hi + hi lo + lo hi in one fp32 accumulator, three instructions for one.
// X, A and B are held 2^12 times as large, which keeps both halves of entries down to 2^-14 of the largest out of fp16's
// subnormal range; entries stay under 2^4, checked on the host from the coefficients.
//
// All operands lie in fragment order (d1_frag.h): a wave's operand of one instruction, 32 rows by 16 of the contraction, is
// one contiguous kilobyte, so loads are whole and LDS tiles are plain copies without conflicts. Rows and columns
// are padded with zeros to 64. A product P Q^T contracts adjacent elements of both: X for A; A (symmetric) for B;
// B and X^T for the new X. So X is kept in both orders and an epilogue writes its tile in both. A and B are symmetric:
// only tiles on and under the diagonal are computed, and written in both places.
// Bound by the matrix units where the matrices are large: a 4,096-wide stack (14.4 TFLOP) has 13.5 ms of products, 1,060
// TFLOP/s (the library's best large product 1,380); eight 1,024 x 1,024 and four 4,096 x 1,024 in halves 780 TFLOP/s of three
// instructions each, whose 384 tiles of 256 take two rounds of 256 CUs; single small matrices by their fifteen
// dependent launches of 5 to 18 us.
#include <math.h>

#include <algorithm>
#include <new>

#include "d1_rows.h"

namespace d1o {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef d1f::floatx16 acc_t;
typedef d1f::u32x4 u32x4;

constexpr int GROUP = 32;                  // matrices of a launch
constexpr int NORM_PARTS = 1024;           // workgroups that sum a matrix's squares (their sums' numbers pass 32 bits from 2^21 matrices on)
constexpr float SCALE = 4096.f;            // of X, A and B as they are held
enum { GRAM, POLY, APPLY, LAST };
enum { C_STEP, C_SKIPPED, C_GO = CTL_GO };

// a matrix as the products see it: m <= n after the turn, M and N their multiples of 64
struct Mat {
    _Float16 *x, *xt[2], *a, *b;           // planes of halves follow each other: hi, then lo
    void *out, *copy;                      // rows x cols as the caller has them
    float size, keep;                      // of a step: out = out * keep - size * O, else out = O
    int32_t rows, cols, m64, n64;
    int32_t splits, first_part;            // workgroups that share a tile's contraction; the first one's partial result
    uint8_t flip, type, step, pad;
};
struct Mats {
    int32_t last[GROUP];                   // workgroups of this and all matrices before, for the launch; past them the largest number
    Mat t[GROUP];
    const int32_t *ctl;
    float *parts;                          // partial results: per workgroup its 32 x 32 blocks as the lanes hold them
    float ca, cb, cc;
    int32_t count, turn;                   // turn: which xt is current
};
// and as its elements come and go
struct Source {
    const void *g;                         // the gradient, or the matrix itself
    float *mom;                            // null: the matrix itself
    _Float16 *x, *xt;
    int32_t rows, cols, m64, n64, parts;
    uint8_t flip, type, pad[2];
};
struct Sources {
    int32_t last[GROUP];
    Source t[GROUP];
    double *sums;                          // [matrix][NORM_PARTS], of the group's first
    double *scales;
    int32_t *parts;                        // how many sums each matrix has
    const int32_t *ctl;
    float mu;
    int32_t count, nesterov;
};

static_assert(sizeof(Mats) <= 4096 && sizeof(Sources) <= 4096, "kernel arguments");

// The matrix of workgroup i: all numbers in one load of kernel arguments, which come from memory (0.7 us each time that one
// load's address waits for another).
__device__ __forceinline__ int find(const int32_t *last, int i, int &within) {
    int k = 0, before = 0;
#pragma unroll
    for (int j = 0; j < GROUP; j++) {
        const int n = last[j];
        k += i >= n;
        before = i >= n ? n : before;
    }
    within = i - before;
    return k;
}

struct Quad {
    float v[4];
};
// four adjacent elements from any address, of which `have` (1 to 4) are there
__device__ __forceinline__ Quad quad(const void *p, int type, int64_t i, int have) {
    Quad q;
    if (type == D1_FP32) {
        const Pack<float, 4> a = load_part<float, 4>((const float *)p + i, have, 0.f);
#pragma unroll
        for (int j = 0; j < 4; j++) q.v[j] = a.v[j];
    } else if (type == D1_BF16) {
        const Pack<__bf16, 4> a = load_part<__bf16, 4>((const __bf16 *)p + i, have, (__bf16)0.f);
#pragma unroll
        for (int j = 0; j < 4; j++) q.v[j] = (float)a.v[j];
    } else {
        const Pack<_Float16, 4> a = load_part<_Float16, 4>((const _Float16 *)p + i, have, (_Float16)0.f);
#pragma unroll
        for (int j = 0; j < 4; j++) q.v[j] = (float)a.v[j];
    }
    return q;
}
// what is orthogonalised, and the new momentum, from the gradient and the momentum before
__device__ __forceinline__ Quad update_of(const Source &t, const Sources &s, Quad g, Quad &m) {
    if (!t.mom) return g;
    Quad u;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        m.v[j] = s.mu * m.v[j] + g.v[j];
        u.v[j] = s.nesterov ? __builtin_fmaf(s.mu, m.v[j], g.v[j]) : m.v[j];
    }
    return u;
}

// sums of squares, a share of the matrix a workgroup; four packs a thread on their way at a time
__global__ __launch_bounds__(256) void k_muon_norm(const Sources s) {
    __shared__ double sh[4];
    int part;
    const int k = find(s.last, blockIdx.x, part);
    const Source &t = s.t[k];
    const int64_t n = (int64_t)t.rows * t.cols, stride = (int64_t)t.parts * 1024;
    double sum = 0.0;
    for (int64_t i = (int64_t)part * 1024 + threadIdx.x * 4; i < n; i += 4 * stride) {
        Quad g[4], m[4];
        int have[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int64_t at = i + u * stride;
            have[u] = n - at >= 4 ? 4 : n - at > 0 ? (int)(n - at) : 0;
            const int64_t from = have[u] ? at : 0;
            g[u] = quad(t.g, t.type, from, have[u]);
            m[u] = t.mom ? quad(t.mom, D1_FP32, from, have[u]) : Quad{};
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const Quad x = update_of(t, s, g[u], m[u]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double d = j < have[u] ? (double)x.v[j] : 0.0;
                sum = __builtin_fma(d, d, sum);
            }
        }
    }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    s.sums[k * NORM_PARTS + part] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
    if (part == 0) s.parts[k] = t.parts;
}

// the matrices' factors; a step whose norms are not all finite is skipped and counted
__global__ __launch_bounds__(1024) void k_muon_begin(const double *__restrict__ sums, double *__restrict__ scales,
                                                     const int32_t *__restrict__ parts, int count, double eps, int32_t *ctl) {
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    for (int k = threadIdx.x >> 6; k < count; k += 16) {
        double sum = 0.0;
        for (int i = threadIdx.x & 63; i < parts[k]; i += 64) sum += sums[(int64_t)k * NORM_PARTS + i];
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
        if ((threadIdx.x & 63) == 0) {
            scales[k] = (double)SCALE / (sqrt(sum) + eps);
            if (!isfinite(sum)) bad = 1;
        }
    }
    __syncthreads();
    if (threadIdx.x || !ctl) return;
    ctl[C_GO] = !bad;
    ctl[bad ? C_SKIPPED : C_STEP]++;
}

__device__ __forceinline__ _Float16 low_half(float v, _Float16 hi) { return (_Float16)(v - (float)hi); }
// elements between the planes of an operand of rows64 x k64 blocks of 64
__device__ __forceinline__ int64_t plane_of(int rows64, int k64) { return (int64_t)rows64 * k64 * 4096; }

// X and X^T in fragment order from 64 x 64 tiles of the update, zeros past its end; the new momentum
template <int TERMS>
__global__ __launch_bounds__(256) void k_muon_prepare(const Sources s) {
    __shared__ __attribute__((aligned(16))) float tile[64][68];
    if (s.ctl && !s.ctl[C_GO]) return;
    int within;
    const int k = find(s.last, blockIdx.x, within);
    const Source &t = s.t[k];
    const double scale = s.scales[k];
    const int cols64 = t.flip ? t.m64 : t.n64;
    const int r0 = within / cols64 * 64, c0 = within % cols64 * 64;
    const int c = c0 + (threadIdx.x & 15) * 4, have = t.cols - c >= 4 ? 4 : t.cols - c > 0 ? t.cols - c : 0;
    Quad g[4], m[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int r = r0 + u * 16 + (threadIdx.x >> 4);
        const int n = r < t.rows ? have : 0;
        const int64_t i = n ? (int64_t)r * t.cols + c : 0;
        g[u] = quad(t.g, t.type, i, n);
        m[u] = t.mom ? quad(t.mom, D1_FP32, i, n) : Quad{};
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int r = r0 + u * 16 + (threadIdx.x >> 4);
        Quad x = update_of(t, s, g[u], m[u]);
        if (t.mom && r < t.rows) {
            Pack<float, 4> out = {{m[u].v[0], m[u].v[1], m[u].v[2], m[u].v[3]}};
            store_part<float, 4>(t.mom + (int64_t)r * t.cols + c, have, out);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) x.v[j] = r < t.rows && j < have ? (float)((double)x.v[j] * scale) : 0.f;
        *(Quad *)&tile[u * 16 + (threadIdx.x >> 4)][(threadIdx.x & 15) * 4] = x;
    }
    __syncthreads();
    // the tile's rows as rows of X (of X^T where the matrix is turned), then its columns as rows of the other
    for (int turn = 0; turn < 2; turn++) {
        const int row64 = (turn ? c0 : r0) >> 6, chunk = (turn ? r0 : c0) >> 6;
        const bool is_x = (turn != 0) == (t.flip != 0);
        _Float16 *out = is_x ? t.x : t.xt;
        const int rows64 = is_x ? t.m64 : t.n64, nch = is_x ? t.n64 : t.m64;
        for (int piece = threadIdx.x; piece < 512; piece += 256) {       // 16 bytes each: 2 row blocks x 4 steps x 64 lanes
            const int rb = piece >> 8, q = piece >> 6 & 3, lane = piece & 63;
            const int row = rb * 32 + (lane & 31), kk = (lane >> 5) * 32 + q * 8;
            half8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = turn ? tile[kk + j][row] : tile[row][kk + j];
                hi[j] = (_Float16)v;
                lo[j] = low_half(v, hi[j]);
            }
            _Float16 *p = out + ((((int64_t)(row64 * 2 + rb) * nch + chunk) * 4 + q) * 64 + lane) * 8;
            *(half8 *)p = hi;
            if (TERMS == 3) *(half8 *)(p + plane_of(rows64, nch)) = lo;
        }
    }
}

// ---- the products

struct Operand {
    const _Float16 *p;
    int64_t plane;
    int rb, k16;              // row blocks of 32, steps of 16
};
struct Job {
    Operand p, q;             // out = p q^T
    int bi, bj;               // tile
    int k_lo, k_hi;           // steps of 16, multiples of 4
    int part;                 // of the launch's partial results
    bool both;                // off the diagonal of a symmetric result: written in both places
};

// the launch's tile `i` of TILE x TILE
template <int MODE, int TILE>
__device__ __forceinline__ int job_of(const Mats &s, int i, Job &job) {
    int within;
    const int k = find(s.last, i, within);
    const Mat &t = s.t[k];
    job.part = t.first_part + within;
    const int split = within % t.splits;
    within /= t.splits;
    const int64_t pm = plane_of(t.m64, t.m64), px = plane_of(t.m64, t.n64);
    job.both = false;
    if (MODE == GRAM || MODE == POLY) {
        job.p = MODE == GRAM ? Operand{t.x, px, t.m64 * 2, t.n64 * 4} : Operand{t.a, pm, t.m64 * 2, t.m64 * 4};
        job.q = job.p;
        int bi = (int)((sqrtf(8.f * within + 1.f) - 1.f) * 0.5f);
        while ((bi + 1) * (bi + 2) / 2 <= within) bi++;
        while (bi * (bi + 1) / 2 > within) bi--;
        job.bi = bi;
        job.bj = within - bi * (bi + 1) / 2;
        job.both = job.bi != job.bj;
    } else {
        job.p = {t.b, pm, t.m64 * 2, t.m64 * 4};
        job.q = {t.xt[s.turn], px, t.n64 * 2, t.m64 * 4};
        if (MODE == LAST && t.flip) {
            const Operand o = job.p;
            job.p = job.q;
            job.q = o;
        }
        const int down = (job.p.rb * 32 + TILE - 1) / TILE;
        job.bi = within % down;
        job.bj = within / down;
    }
    const int chunks = job.p.k16 / 4, per = (chunks + t.splits - 1) / t.splits;
    job.k_lo = split * per * 4;
    job.k_hi = (split * per + per < chunks ? split * per + per : chunks) * 4;
    return k;
}

__device__ __forceinline__ acc_t mma(half8 a, half8 b, acc_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// The block of A that POLY's result needs, as the lanes hold the result
struct Held {
    half4 hi[4], lo[4];
};
__device__ __forceinline__ int64_t natural(int nch, int I, int J) {
    const int lane = threadIdx.x & 63;
    return ((((int64_t)J * nch + (I >> 1)) * 4) * 64 + (lane & 31) + 32 * (I & 1)) * 8 + 4 * (lane >> 5);
}
template <int MODE, int TERMS>
__device__ __forceinline__ Held held_of(const Mats &s, const Mat &t, const Job &job, int I, int J) {
    Held h = {};
    if (MODE != POLY || I >= job.p.rb || J >= job.q.rb) return h;
    const int64_t at = natural(t.m64, I, J), plane = plane_of(t.m64, t.m64);
#pragma unroll
    for (int g = 0; g < 4; g++) {
        h.hi[g] = *(const half4 *)(t.a + at + g * 512);
        if (TERMS == 3) h.lo[g] = *(const half4 *)(t.a + plane + at + g * 512);
    }
    return h;
}

// A result's last form: O itself, or the parameter's step; all of the parameter's loads before the first store
template <class T>
__device__ __forceinline__ void put_last(T *out, const Mat &t, acc_t d, int64_t at, int rows) {
    constexpr float DOWN = 1.f / (SCALE * SCALE);
    T p[16];
    if (t.step)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int row = d1f::drow(r, 0);
            p[r] = row < rows ? out[at + (int64_t)row * t.cols] : (T)0.f;
        }
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int row = d1f::drow(r, 0);
        const float o = d[r] * DOWN, v = t.step ? (float)p[r] * t.keep - t.size * o : o;
        if (row < rows) {
            out[at + (int64_t)row * t.cols] = (T)v;
            if (t.copy) ((__bf16 *)t.copy)[at + (int64_t)row * t.cols] = (__bf16)v;
        }
    }
}

// A 32 x 32 result: lane l of register r holds row 8 (r / 4) + 4 (l / 32) + r % 4 of block I, column l % 32 of block J.
// `scratch`: the wave's 32 x 40 halves of LDS.
template <int MODE, int TERMS>
__device__ __forceinline__ void put_tile(const Mats &s, const Mat &t, const Job &job, acc_t d, const Held &held, int I, int J,
                                         _Float16 *scratch) {
    const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
    if (I >= job.p.rb || J >= job.q.rb) return;              // the whole wave
    if (MODE == LAST) {
        const int c = J * 32 + col;
        if (c >= t.cols) return;
        const int64_t at = (int64_t)(I * 32 + 4 * h) * t.cols + c;
        const int rows = t.rows - I * 32 - 4 * h;            // of this lane's first row's on
        if (t.type == D1_FP32)
            put_last((float *)t.out, t, d, at, rows);
        else if (t.type == D1_BF16)
            put_last((__bf16 *)t.out, t, d, at, rows);
        else
            put_last((_Float16 *)t.out, t, d, at, rows);
        return;
    }
    _Float16 *to = MODE == GRAM ? t.a : MODE == POLY ? t.b : t.xt[s.turn ^ 1];      // rows J, contraction I
    const int nch = t.m64;
    const int64_t plane = MODE == APPLY ? plane_of(t.m64, t.n64) : plane_of(t.m64, t.m64);
    const int64_t at = natural(nch, I, J);
    half4 hi[4], lo[4];
#pragma unroll
    for (int g = 0; g < 4; g++) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = d[4 * g + j] * (1.f / SCALE);
        if (MODE == POLY) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float a = TERMS == 3 ? (float)held.hi[g][j] + (float)held.lo[g][j] : (float)held.hi[g][j];
                v[j] = __builtin_fmaf(s.cc, v[j], s.cb * a);
                if (I == J && 8 * g + 4 * h + j == col) v[j] += s.ca * SCALE;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            hi[g][j] = (_Float16)v[j];
            lo[g][j] = low_half(v[j], hi[g][j]);
        }
        *(half4 *)(to + at + g * 512) = hi[g];
        if (TERMS == 3) *(half4 *)(to + plane + at + g * 512) = lo[g];
    }
    if (MODE != APPLY && !job.both) return;
    // the other order: rows I, contraction J
    if (MODE == APPLY) to = t.x;
    const int nch2 = MODE == APPLY ? t.n64 : t.m64;
#pragma unroll
    for (int p = 0; p < (TERMS == 3 ? 2 : 1); p++) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) scratch[(8 * g + 4 * h + j) * 40 + col] = p ? lo[g][j] : hi[g][j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int q = h + 2 * e;
            const half8 v = *(const half8 *)(scratch + col * 40 + q * 8);
            *(half8 *)(to + p * plane + ((((int64_t)I * nch2 + (J >> 1)) * 4 + q) * 64 + col + 32 * (J & 1)) * 8) = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
}

// A share of a tile's contraction: the wave's 32 x 32 block `at` of `blocks`, as the lanes hold it
__device__ __forceinline__ void put_part(const Mats &s, const Mat &, const Job &job, acc_t d, int blocks, int at) {
    float *p = s.parts + ((int64_t)job.part * blocks + at) * 1024 + (threadIdx.x & 63) * 4;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const Pack<float, 4> v = {{d[4 * g], d[4 * g + 1], d[4 * g + 2], d[4 * g + 3]}};
        store<float, 4>(p + g * 256, v);
    }
}
// and the shares joined, in their order: a wave a block
template <int MODE, int TERMS, int TILE>
__global__ __launch_bounds__(256) void k_muon_join(const Mats s) {
    constexpr int RB = TILE / 32, BLOCKS = RB * RB;
    __shared__ __attribute__((aligned(16))) _Float16 scratch[4][32 * 40];
    if (s.ctl && !s.ctl[C_GO]) return;
    const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = (int)(id / BLOCKS), at = (int)(id % BLOCKS);
    // tiles of the matrices whose contraction is shared; the others were finished where they were made
    int k = 0, left = tile;
    for (; k < s.count; k++) {
        const int tiles = s.t[k].splits > 1 ? (s.last[k] - (k ? s.last[k - 1] : 0)) / s.t[k].splits : 0;
        if (left < tiles) break;
        left -= tiles;
    }
    if (k == s.count) return;
    const Mat &t = s.t[k];
    Job job;
    job_of<MODE, TILE>(s, (k ? s.last[k - 1] : 0) + left * t.splits, job);
    const Held held = held_of<MODE, TERMS>(s, t, job, job.bi * RB + at / RB, job.bj * RB + at % RB);
    acc_t d;
#pragma unroll
    for (int r = 0; r < 16; r++) d[r] = 0.f;
    for (int w = 0; w < t.splits; w++) {
        const float *p = s.parts + ((int64_t)(job.part + w) * BLOCKS + at) * 1024 + (threadIdx.x & 63) * 4;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const Pack<float, 4> v = load<float, 4>(p + g * 256);
#pragma unroll
            for (int j = 0; j < 4; j++) d[4 * g + j] += v.v[j];
        }
    }
    put_tile<MODE, TERMS>(s, t, job, d, held, job.bi * RB + at / RB, job.bj * RB + at % RB, scratch[threadIdx.x >> 6]);
}

// Small results: a workgroup a tile of 32 SIDE, its waves share the contraction and join in LDS; operands straight from
// the caches into registers; other workgroups of the CU multiply while one loads (with the next operands on their way there
// were half as many: 544 tiles of 32 with a contraction of 256 in two halves 11.3 us, 7.8 without).
template <int MODE, int TERMS, int SIDE, int W>
__global__ __launch_bounds__(64 * W) void k_muon_small(const Mats s) {
    constexpr int PL = TERMS == 3 ? 2 : 1, AT_ONCE = TERMS == 3 && SIDE == 2 ? 2 : 4;
    __shared__ float sums[W][SIDE * SIDE][16][64];
    if (s.ctl && !s.ctl[C_GO]) return;
    Job job;
    const Mat &t = s.t[job_of<MODE, 32 * SIDE>(s, blockIdx.x, job)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    acc_t acc[SIDE][SIDE];
#pragma unroll
    for (int i = 0; i < SIDE; i++)
#pragma unroll
        for (int j = 0; j < SIDE; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
    const _Float16 *p[SIDE], *q[SIDE];
#pragma unroll
    for (int i = 0; i < SIDE; i++) {
        const int I = job.bi * SIDE + i, J = job.bj * SIDE + i;
        p[i] = job.p.p + (int64_t)(I < job.p.rb ? I : job.p.rb - 1) * job.p.k16 * 512 + lane * 8;
        q[i] = job.q.p + (int64_t)(J < job.q.rb ? J : job.q.rb - 1) * job.q.k16 * 512 + lane * 8;
    }
    const int first = job.k_lo / AT_ONCE, batches = job.k_hi / AT_ONCE, per = (batches - first + W - 1) / W;      // multiples of 4
    const int lo = first + wave * per, hi = lo + per < batches ? lo + per : batches;
    Held held = {};
    if (wave < SIDE * SIDE) held = held_of<MODE, TERMS>(s, t, job, job.bi * SIDE + wave / SIDE, job.bj * SIDE + wave % SIDE);
    for (int c = lo; c < hi; c++) {
        half8 a[AT_ONCE][PL][SIDE], b[AT_ONCE][PL][SIDE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; k++)
#pragma unroll
            for (int pl = 0; pl < PL; pl++)
#pragma unroll
                for (int i = 0; i < SIDE; i++) {
                    a[k][pl][i] = *(const half8 *)(p[i] + pl * job.p.plane + (c * AT_ONCE + k) * 512);
                    b[k][pl][i] = *(const half8 *)(q[i] + pl * job.q.plane + (c * AT_ONCE + k) * 512);
                }
#pragma unroll
        for (int k = 0; k < AT_ONCE; k++)
#pragma unroll
            for (int i = 0; i < SIDE; i++)
#pragma unroll
                for (int j = 0; j < SIDE; j++) {
                    acc[i][j] = mma(a[k][0][i], b[k][0][j], acc[i][j]);
                    if (TERMS == 3) {
                        acc[i][j] = mma(a[k][0][i], b[k][PL - 1][j], acc[i][j]);
                        acc[i][j] = mma(a[k][PL - 1][i], b[k][0][j], acc[i][j]);
                    }
                }
    }
#pragma unroll
    for (int i = 0; i < SIDE; i++)
#pragma unroll
        for (int j = 0; j < SIDE; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) sums[wave][i * SIDE + j][r][lane] = acc[i][j][r];
    __syncthreads();
    acc_t d;
    if (wave < SIDE * SIDE)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            float x[W];
#pragma unroll
            for (int w = 0; w < W; w++) x[w] = sums[w][wave][r][lane];
            d[r] = (x[0] + x[1]) + (x[2] + x[3]);
            if constexpr (W == 8) d[r] += (x[4] + x[5]) + (x[6] + x[7]);
        }
    __syncthreads();
    if (wave >= SIDE * SIDE) return;
    if (t.splits > 1)
        put_part(s, t, job, d, SIDE * SIDE, wave);
    else
        put_tile<MODE, TERMS>(s, t, job, d, held, job.bi * SIDE + wave / SIDE, job.bj * SIDE + wave % SIDE, (_Float16 *)sums[wave]);
}

// Large results: a workgroup a tile of TILE x TILE, operands through a ring of LDS buffers that memory fills directly:
// while one is multiplied, three more are on their way (with one ahead the matrix units idled nearly half the time: a
// stage's products are over before the next stage's loads from the last cache).
constexpr int waves_of(int tile) { return tile == 256 ? 8 : 4; }
template <int TERMS, int TILE>
struct Large {
    static constexpr int WAVES = waves_of(TILE);
    static constexpr int DOWN = 2, ACROSS = WAVES / 2;                    // waves
    static constexpr int NI = TILE / 32 / DOWN, NJ = TILE / 32 / ACROSS;  // results a wave
    static constexpr int PL = TERMS == 3 ? 2 : 1, RB = TILE / 32;
    static constexpr int QS = TERMS == 3 ? 1 : 2;                         // steps of 16 a stage
    static constexpr int PIECES = 2 * PL * RB * QS;                       // kilobytes a stage
    static constexpr int MINE = PIECES / WAVES;                           // a wave's
    static constexpr int STAGE = PIECES * 512;                            // halves
    static constexpr int RING = 4;
};
typedef __attribute__((address_space(3))) void lds_void;

// All but the last LEFT of this wave's loads have landed and its LDS reads are done; then the workgroup's.
template <int LEFT>
__device__ __forceinline__ void wait_stage() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// (apart from the kernel, whose host side does not know buffer descriptors)
template <int MODE, int TERMS, int TILE>
__device__ __forceinline__ void large_tile(const Mats &s) {
    typedef Large<TERMS, TILE> L;
    __shared__ __attribute__((aligned(16))) _Float16 lds[L::RING][L::STAGE];
    if (s.ctl && !s.ctl[C_GO]) return;
    Job job;
    const Mat &t = s.t[job_of<MODE, TILE>(s, blockIdx.x, job)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wi = wave / L::ACROSS, wj = wave % L::ACROSS;
    acc_t acc[L::NI][L::NJ];
#pragma unroll
    for (int i = 0; i < L::NI; i++)
#pragma unroll
        for (int j = 0; j < L::NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
    // kilobyte e of a stage: operand, plane, row block, step. (Buffer loads: behind global loads to LDS the compiler
    // waits for all LDS reads where it needs the earlier ones alone.)
    __amdgpu_buffer_rsrc_t from[L::MINE];
#pragma unroll
    for (int e = 0; e < L::MINE; e++) {
        const int piece = e * L::WAVES + wave, k = piece % L::QS, rb = piece / L::QS % L::RB, pl = piece / (L::QS * L::RB) % L::PL,
                  side = piece / (L::QS * L::RB * L::PL);
        const Operand &o = side ? job.q : job.p;
        int R = (side ? job.bj : job.bi) * L::RB + rb;
        if (R >= o.rb) R = o.rb - 1;
        from[e] = __builtin_amdgcn_make_buffer_rsrc((void *)(o.p + pl * o.plane + ((int64_t)R * o.k16 + job.k_lo + k) * 512), 0,
                                                    (o.k16 - job.k_lo - k) * 1024, 0x00020000);
    }
    auto fetch = [&](int stage) {
#pragma unroll
        for (int e = 0; e < L::MINE; e++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from[e], (lds_void *)(lds[stage % L::RING] + (e * L::WAVES + wave) * 512), 16,
                                                     lane * 16, stage * L::QS * 1024, 0, 0);
    };
    // A step's operands are read while the step before is multiplied, also into the next stage: by its barrier every wave has
    // read all of the stage before, whose buffer is then filled again.
    half8 a[2][L::PL][L::NI], b[2][L::PL][L::NJ];
    auto operands = [&](int step, int to) {
        const _Float16 *at = lds[step / L::QS % L::RING] + step % L::QS * 512 + lane * 8;
        const _Float16 *a0 = at + wi * L::NI * L::QS * 512, *b0 = at + (L::PL * L::RB + wj * L::NJ) * L::QS * 512;
#pragma unroll
        for (int pl = 0; pl < L::PL; pl++) {
#pragma unroll
            for (int i = 0; i < L::NI; i++) a[to][pl][i] = *(const half8 *)(a0 + (pl * L::RB + i) * L::QS * 512);
#pragma unroll
            for (int j = 0; j < L::NJ; j++) b[to][pl][j] = *(const half8 *)(b0 + (pl * L::RB + j) * L::QS * 512);
        }
    };
    const int steps = job.k_hi - job.k_lo, stages = steps / L::QS;       // steps: a multiple of 4
    for (int st = 0; st < L::RING && st < stages; st++) fetch(st);
    if (L::RING - 1 < stages)
        wait_stage<(L::RING - 1) * L::MINE>();
    else
        wait_stage<0>();
    operands(0, 0);
    auto multiply = [&](int of) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < L::NI; i++)
#pragma unroll
            for (int j = 0; j < L::NJ; j++) {
                acc[i][j] = mma(a[of][0][i], b[of][0][j], acc[i][j]);
                if (TERMS == 3) {
                    acc[i][j] = mma(a[of][0][i], b[of][L::PL - 1][j], acc[i][j]);
                    acc[i][j] = mma(a[of][L::PL - 1][i], b[of][0][j], acc[i][j]);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    // without conditions as long as there is a stage to fetch, so that the waits are those of one path
    int g = 0;
    for (; (g + 4) / L::QS + L::RING - 1 < stages; g += 4) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int next = g + u + 1;
            if ((u + 1) % L::QS == 0) {
                wait_stage<(L::RING - 2) * L::MINE>();
                fetch(next / L::QS + L::RING - 1);
            }
            operands(next, (u + 1) & 1);
            multiply(u & 1);
        }
    }
    for (; g < steps; g += 4) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int next = g + u + 1;
            if ((u + 1) % L::QS == 0 && next < steps) {
                wait_stage<0>();
                if (next / L::QS + L::RING - 1 < stages) fetch(next / L::QS + L::RING - 1);
            }
            operands(next, (u + 1) & 1);       // behind the last step something that is not used
            multiply(u & 1);
        }
    }
    wait_stage<0>();                       // the ring becomes the waves' scratch
    _Float16 *scratch = lds[0] + wave * 32 * 40;
#pragma unroll
    for (int i = 0; i < L::NI; i++)
#pragma unroll
        for (int j = 0; j < L::NJ; j++) {
            const int I = wi * L::NI + i, J = wj * L::NJ + j;
            if (t.splits > 1)
                put_part(s, t, job, acc[i][j], L::RB * L::RB, I * L::RB + J);
            else
                put_tile<MODE, TERMS>(s, t, job, acc[i][j], held_of<MODE, TERMS>(s, t, job, job.bi * L::RB + I, job.bj * L::RB + J), job.bi * L::RB + I,
                                job.bj * L::RB + J, scratch);
        }
}
template <int MODE, int TERMS, int TILE>
__global__ __launch_bounds__(64 * waves_of(TILE)) void k_muon_large(const Mats s) {
    large_tile<MODE, TERMS, TILE>(s);
}

// ---- the host's side

inline int up64(int64_t x) { return (int)((x + 63) / 64); }
struct Shape {
    int m64, n64;
    bool flip;
};
inline Shape shape_of(const D1MuonTensor &t) {
    const bool flip = t.rows > t.cols;
    return {up64(flip ? t.cols : t.rows), up64(flip ? t.rows : t.cols), flip};
}
// bytes of a matrix's operands: X and two X^T, A and B
inline int64_t mat_bytes(const D1MuonTensor &t, int terms) {
    const Shape h = shape_of(t);
    const int64_t planes = terms == 3 ? 2 : 1;
    return planes * 8192 * (3 * (int64_t)h.m64 * h.n64 + 2 * (int64_t)h.m64 * h.m64);
}
constexpr int64_t GROUP_BYTES = (int64_t)4 << 30;
// Kinds of kernels: small tiles of 32 and 64, large ones of 128 (two workgroups a CU) and of 256
enum { SMALL32, SMALL64, LARGE128, LARGE256, KINDS };
constexpr int side_of(int kind) { return kind == SMALL32 ? 32 : kind == SMALL64 ? 64 : kind == LARGE256 ? 256 : 128; }
inline int64_t tiles_of(int mode, const Shape &h, int side) {
    const int64_t m = ((int64_t)h.m64 * 64 + side - 1) / side, n = ((int64_t)h.n64 * 64 + side - 1) / side;
    return mode == GRAM || mode == POLY ? m * (m + 1) / 2 : m * n;
}
// With a short side under 16 an entry of A weighs a whole row or more, and its rounding moves all of it: in 16-bit operands the worst of
// 300 random 2 x 2 matrices is 4.4% off, of 4 x 300 0.7% (32 x 32 0.25%; bf16's own rounding of the result 0.16%). Two halves take that away,
// for 8 x 256 90 us in place of 78 and 15 x 131,072 618 for 267; in a list with others that stay in 16 bits, a second row of
// launches (eight 8 x 256 beside eight 1,024 x 1,024 538 us, 453).
inline int terms_of(const D1MuonTensor &t, const D1Muon *h) {
    if (h->terms) return h->terms;
    return t.type == D1_FP32 || t.rows < 16 || t.cols < 16 ? 3 : 1;
}
// The matrices at[from..to) that one row of launches takes: alike in terms, as many as fit its arguments and 4 GB
inline int group_end(const D1MuonTensor *t, const int *at, int count, int from, const D1Muon *h) {
    const int terms = terms_of(t[at[from]], h);
    int64_t bytes = 0;
    int to = from;
    while (to < count && to - from < GROUP && terms_of(t[at[to]], h) == terms) {
        bytes += mat_bytes(t[at[to]], terms);
        if (to > from && bytes > GROUP_BYTES) break;
        to++;
    }
    return to;
}
inline int parts_of(const D1MuonTensor &t) {
    const int64_t n = (t.rows * t.cols + 4095) / 4096;
    return (int)(n < 1 ? 1 : n < NORM_PARTS ? n : NORM_PARTS);
}
// How a launch shares its products: the kind of tile and how many steps of 64 of the contraction a workgroup takes at most.
// The estimate, in us: a kind's time for 64 of a tile's contraction where it has its CU full (WORK; the largest tiles, one
// to a CU, in rounds) and alone (ALONE), and for shared tiles the join's launch and bytes at 4 TB/s.
// steps of 64 above which eight waves share a small tile's contraction, not four (a matrix's product with itself: 256 x 1,800 in
// halves by tiles of 32 10.8 us, 13.4 by four waves; 1,000 x 4,001 by tiles of 64 18.2, 24.0)
constexpr int WIDE = 12;
struct Plan {
    int kind;
    int64_t most;             // steps of 64
};
inline int64_t chunks_of(int mode, const Shape &h) { return mode == GRAM ? h.n64 : h.m64; }
inline int64_t splits_of(int64_t chunks, int64_t most) { return (chunks + most - 1) / most; }
struct Alike {
    Shape h;
    int n;
};
static double plan_time(const Alike *shapes, int count, int mode, int terms, int kind, int64_t most) {
    static const double WORK[2][KINDS] = {{0.117, 0.38, 0.68, 1.75}, {0.26, 0.87, 1.95, 5.3}},
                        ALONE[2][KINDS] = {{0.15, 0.3, 0.9, 1.75}, {0.32, 0.6, 2.2, 5.3}};
    double c = WORK[terms == 3][kind], l = ALONE[terms == 3][kind];
    double work = 0, groups = 0, longest = 0, joined = 0;
    for (int k = 0; k < count; k++) {
        const Shape &h = shapes[k].h;
        const int64_t chunks = chunks_of(mode, h), splits = splits_of(chunks, most), each = (chunks + splits - 1) / splits;
        const double n = (double)tiles_of(mode, h, side_of(kind)) * splits * shapes[k].n;
        work += n * each;
        groups += n;
        if (each > longest) longest = (double)each;
        if (splits > 1) joined += n * side_of(kind) * side_of(kind) * 8;
    }
    if (kind <= SMALL64 && longest > WIDE) c *= 1.4, l *= 0.7;
    double time = work * c / 256;
    const double rounds = std::ceil(groups / 256) * work / groups;
    if (kind == LARGE256 && rounds * c > time) time = rounds * c;
    if (longest * l > time) time = longest * l;
    return time + (joined ? 9.0 + joined / 4e6 : 0.0);
}
static Plan plan_of(const D1MuonTensor *t, const int *at, int count, int mode, int terms) {
    Alike shapes[GROUP];
    int alike = 0;
    int64_t longest = 0;
    for (int k = 0; k < count; k++) {
        const Shape h = shape_of(t[at[k]]);
        if (chunks_of(mode, h) > longest) longest = chunks_of(mode, h);
        int i = 0;
        while (i < alike && (shapes[i].h.m64 != h.m64 || shapes[i].h.n64 != h.n64)) i++;
        if (i == alike) shapes[alike++] = {h, 0};
        shapes[i].n++;
    }
    Plan best{0, 1 << 20};
    double least = 1e30;
    for (int kind = 0; kind < KINDS; kind++)
        for (int64_t most : {(int64_t)1 << 20, (int64_t)64, (int64_t)32, (int64_t)16, (int64_t)8, (int64_t)4}) {
            if (most < (1 << 20) && (most >= longest || mode == APPLY)) continue;
            const double time = plan_time(shapes, alike, mode, terms, kind, most);
            if (time < least) {
                least = time;
                best = {kind, most};
            }
        }
    return best;
}
// bytes of a launch's partial results
static int64_t plan_bytes(const D1MuonTensor *t, const int *at, int count, int mode, const Plan &p) {
    int64_t bytes = 0;
    for (int k = 0; k < count; k++) {
        const Shape h = shape_of(t[at[k]]);
        const int64_t splits = splits_of(chunks_of(mode, h), p.most);
        if (splits > 1) bytes += tiles_of(mode, h, side_of(p.kind)) * splits * side_of(p.kind) * side_of(p.kind) * 4;
    }
    return bytes;
}

// The singular values of X lie in [0, 1] after the norm; the largest that the steps make of them, from the ends and the
// turning points of a s + b s^3 + c s^5 and of its factor a + b s^2 + c s^4. What is held has to stay under 2^4 times the scale.
static double reach_of(const D1Muon *h) {
    double top = 1.0;
    for (int k = 0; k < h->steps; k++) {
        const double x1 = top * top;
        double x[5] = {0.0, x1, x1, x1, x1};               // s^2
        if (h->c != 0) {
            x[2] = -h->b / (2 * h->c);
            const double d = 9 * h->b * h->b - 20 * h->a * h->c;
            if (d >= 0) {
                x[3] = (-3 * h->b + sqrt(d)) / (10 * h->c);
                x[4] = (-3 * h->b - sqrt(d)) / (10 * h->c);
            }
        } else if (h->b != 0) {
            x[3] = -h->a / (3 * h->b);
        }
        double most = 0.0;
        for (double at : x) {
            if (!(at > 0)) at = 0;
            if (at > x1) at = x1;
            const double factor = fabs(h->a + h->b * at + h->c * at * at);
            if (!(factor < 15.0)) return INFINITY;
            if (factor * sqrt(at) > most) most = factor * sqrt(at);
        }
        top = most + 1e-3;
        if (!(top < 3.8)) return INFINITY;
    }
    return top;
}

static bool muon_args(const D1MuonTensor *t, int count, const D1Muon *h) {
    if (count < 0 || (count && !t) || !h || (h->terms != 0 && h->terms != 1 && h->terms != 3) || h->part < 0 || h->part > 2) return false;
    if (h->steps < 1 || h->steps > D1_MUON_MAX_STEPS || !(h->eps >= 0) || !(h->momentum >= 0 && h->momentum < 1)) return false;
    for (int i = 0; i < count; i++) {
        const D1MuonTensor &a = t[i];
        if (a.rows < 0 || a.cols < 0 || a.rows > D1_MUON_MAX_SIDE || a.cols > D1_MUON_MAX_SIDE) return false;
        if (a.rows == 0 || a.cols == 0) continue;
        if (!is_type(a.gtype) || !is_type(a.type) || !a.g || !a.out || !(a.lr - a.lr == 0) || !(a.weight_decay - a.weight_decay == 0)) return false;
        if (a.momentum && (a.type == D1_FP16 || a.gtype == D1_FP16)) return false;
        if (!a.momentum && a.copy) return false;
    }
    return true;
}

// the matrices with elements, in the order of the launches: alike in terms, the longest products first, so that none
// starts when the others are over
static int muon_order(const D1MuonTensor *t, int count, const D1Muon *h, int *at) {
    int live = 0;
    for (int i = 0; i < count; i++)
        if (t[i].rows && t[i].cols) at[live++] = i;
    auto longest = [&](int i) { return terms_of(t[i], h) * (int64_t)1000000 + (t[i].rows > t[i].cols ? t[i].rows : t[i].cols); };
    std::stable_sort(at, at + live, [&](int x, int y) { return longest(x) > longest(y); });
    return live;
}
struct MuonWork {
    int64_t parts, sums, scales, mats, shares, total;    // offsets: sums' counts, sums, factors, a group's operands, partial results
};
static MuonWork muon_work(const D1MuonTensor *t, int count, const D1Muon *h, const int *at, int live) {
    MuonWork w;
    w.parts = 0;
    w.sums = ((int64_t)count * 4 + 255) & ~(int64_t)255;
    w.scales = w.sums + (int64_t)count * NORM_PARTS * 8;
    w.mats = (w.scales + (int64_t)count * 8 + 255) & ~(int64_t)255;
    int64_t most = 0, shares = 0;
    for (int from = 0, to; from < live; from = to) {
        to = group_end(t, at, live, from, h);
        const int terms = terms_of(t[at[from]], h);
        int64_t bytes = 0;
        for (int k = from; k < to; k++) bytes += mat_bytes(t[at[k]], terms);
        most = bytes > most ? bytes : most;
        for (int mode : {(int)GRAM, (int)POLY, (int)APPLY}) {
            const int64_t b = plan_bytes(t, at + from, to - from, mode, plan_of(t, at + from, to - from, mode, terms));
            shares = b > shares ? b : shares;
        }
    }
    w.shares = w.mats + most;
    w.total = w.shares + shares;
    return w;
}

// `groups` workgroups; `blocks`: 32 x 32 blocks of tiles whose contraction is shared (of A and B alone)
template <int MODE, int TERMS>
static void muon_products(const Mats &s, int kind, bool wide, int64_t groups, int64_t blocks, hipStream_t stream) {
    const dim3 grid((unsigned)groups), block(256), joins((unsigned)((blocks + 3) / 4));
    if (kind == LARGE256)
        hipLaunchKernelGGL((k_muon_large<MODE, TERMS, 256>), grid, dim3(512), 0, stream, s);
    else if (kind == LARGE128)
        hipLaunchKernelGGL((k_muon_large<MODE, TERMS, 128>), grid, block, 0, stream, s);
    else if (kind == SMALL64 && wide)
        hipLaunchKernelGGL((k_muon_small<MODE, TERMS, 2, 8>), grid, dim3(512), 0, stream, s);
    else if (kind == SMALL64)
        hipLaunchKernelGGL((k_muon_small<MODE, TERMS, 2, 4>), grid, block, 0, stream, s);
    else if (wide)
        hipLaunchKernelGGL((k_muon_small<MODE, TERMS, 1, 8>), grid, dim3(512), 0, stream, s);
    else
        hipLaunchKernelGGL((k_muon_small<MODE, TERMS, 1, 4>), grid, block, 0, stream, s);
    if constexpr (MODE == GRAM || MODE == POLY) {
        if (!blocks) return;
        if (kind == LARGE256)
            hipLaunchKernelGGL((k_muon_join<MODE, TERMS, 256>), joins, block, 0, stream, s);
        else if (kind == LARGE128)
            hipLaunchKernelGGL((k_muon_join<MODE, TERMS, 128>), joins, block, 0, stream, s);
        else if (kind == SMALL64)
            hipLaunchKernelGGL((k_muon_join<MODE, TERMS, 64>), joins, block, 0, stream, s);
        else
            hipLaunchKernelGGL((k_muon_join<MODE, TERMS, 32>), joins, block, 0, stream, s);
    }
}
template <int TERMS>
static void muon_products(int mode, const Mats &s, int kind, bool wide, int64_t groups, int64_t blocks, hipStream_t stream) {
    if (mode == GRAM)
        muon_products<GRAM, TERMS>(s, kind, wide, groups, blocks, stream);
    else if (mode == POLY)
        muon_products<POLY, TERMS>(s, kind, wide, groups, blocks, stream);
    else if (mode == APPLY)
        muon_products<APPLY, TERMS>(s, kind, wide, groups, blocks, stream);
    else
        muon_products<LAST, TERMS>(s, kind, wide, groups, blocks, stream);
}

static int muon_run(const D1MuonTensor *t, const D1Muon *h, int32_t *ctl, char *work, const MuonWork &w, const int *at, int live,
                    hipStream_t stream) {
    double *sums = (double *)(work + w.sums), *scales = (double *)(work + w.scales);
    int32_t *parts = (int32_t *)(work + w.parts);
    auto sources = [&](int from, int to, bool prepare, Sources &s) {
        s = Sources{};
        for (int32_t &n : s.last) n = INT32_MAX;
        s.sums = sums + (int64_t)from * NORM_PARTS;
        s.scales = scales + from;
        s.parts = parts + from;
        s.ctl = ctl;
        s.mu = (float)h->momentum;
        s.nesterov = h->nesterov;
        int64_t tiles = 0;
        for (int k = from; k < to; k++) {
            const D1MuonTensor &a = t[at[k]];
            const Shape sh = shape_of(a);
            Source &o = s.t[s.count++];
            o.g = a.g;
            o.mom = a.momentum;
            o.rows = (int32_t)a.rows;
            o.cols = (int32_t)a.cols;
            o.m64 = sh.m64;
            o.n64 = sh.n64;
            o.flip = sh.flip;
            o.type = a.gtype;
            o.parts = parts_of(a);
            tiles += prepare ? (int64_t)sh.m64 * sh.n64 : o.parts;
            s.last[s.count - 1] = (int32_t)tiles;
        }
        return tiles;
    };
    if (h->part != 2) {
        for (int from = 0; from < live;) {
            const int to = live - from < GROUP ? live : from + GROUP;
            Sources s;
            const int64_t tiles = sources(from, to, false, s);
            hipLaunchKernelGGL(k_muon_norm, dim3((unsigned)tiles), dim3(256), 0, stream, s);
            from = to;
        }
        hipLaunchKernelGGL(k_muon_begin, dim3(1), dim3(1024), 0, stream, sums, scales, parts, live, h->eps, ctl);
    }
    if (h->part == 1) return (int)hipGetLastError();
    for (int from = 0; from < live;) {
        const int to = group_end(t, at, live, from, h), terms = terms_of(t[at[from]], h);
        Sources s;
        const int64_t tiles = sources(from, to, true, s);
        Mats p{};
        for (int32_t &n : p.last) n = INT32_MAX;
        p.ctl = ctl;
        p.ca = (float)h->a;
        p.cb = (float)h->b;
        p.cc = (float)h->c;
        p.count = to - from;
        _Float16 *free = (_Float16 *)(work + w.mats);
        const int planes = terms == 3 ? 2 : 1;
        for (int k = 0; k < p.count; k++) {
            const D1MuonTensor &a = t[at[from + k]];
            const Shape sh = shape_of(a);
            const int64_t px = (int64_t)sh.m64 * sh.n64 * 4096 * planes, pm = (int64_t)sh.m64 * sh.m64 * 4096 * planes;
            Mat &o = p.t[k];
            o.x = free;
            o.xt[0] = o.x + px;
            o.xt[1] = o.xt[0] + px;
            o.a = o.xt[1] + px;
            o.b = o.a + pm;
            free = o.b + pm;
            o.out = a.out;
            o.copy = a.copy;
            o.step = a.momentum != nullptr;
            o.size = (float)(a.lr * a.scale);
            o.keep = (float)(1.0 - a.lr * a.weight_decay);
            o.rows = (int32_t)a.rows;
            o.cols = (int32_t)a.cols;
            o.m64 = sh.m64;
            o.n64 = sh.n64;
            o.flip = sh.flip;
            o.type = a.type;
            s.t[k].x = o.x;
            s.t[k].xt = o.xt[0];
        }
        if (terms == 3)
            hipLaunchKernelGGL(k_muon_prepare<3>, dim3((unsigned)tiles), dim3(256), 0, stream, s);
        else
            hipLaunchKernelGGL(k_muon_prepare<1>, dim3((unsigned)tiles), dim3(256), 0, stream, s);
        p.parts = (float *)(work + w.shares);
        Plan plans[3];
        for (int mode : {(int)GRAM, (int)POLY, (int)APPLY}) plans[mode] = plan_of(t, at + from, p.count, mode, terms);
        for (int step = 0; step < h->steps; step++) {
            p.turn = step & 1;
            for (int mode : {(int)GRAM, (int)POLY, step + 1 < h->steps ? (int)APPLY : (int)LAST}) {
                const Plan &plan = plans[mode == LAST ? (int)APPLY : mode];
                const int side = side_of(plan.kind);
                int64_t groups = 0, parts = 0, blocks = 0, longest = 0;
                for (int k = 0; k < p.count; k++) {
                    const Shape sh = shape_of(t[at[from + k]]);
                    const int64_t chunks = chunks_of(mode, sh), tiles = tiles_of(mode, sh, side);
                    int64_t splits = splits_of(chunks, plan.most);
                    splits = splits_of(chunks, (chunks + splits - 1) / splits);       // none without a step
                    p.t[k].splits = (int32_t)splits;
                    longest = std::max(longest, (chunks + splits - 1) / splits);
                    p.t[k].first_part = (int32_t)parts;
                    groups += tiles * splits;
                    if (splits > 1) {
                        parts += tiles * splits;
                        blocks += tiles * (side / 32) * (side / 32);
                    }
                    p.last[k] = (int32_t)groups;
                }
                if (terms == 3)
                    muon_products<3>(mode, p, plan.kind, longest > WIDE, groups, blocks, stream);
                else
                    muon_products<1>(mode, p, plan.kind, longest > WIDE, groups, blocks, stream);
            }
        }
        from = to;
    }
    return (int)hipGetLastError();
}

}  // namespace d1o

using namespace d1o;

extern "C" {
int64_t d1_muon_work_bytes(const D1MuonTensor *t, int count, const D1Muon *h) {
    if (!muon_args(t, count, h)) return D1_E_ARG;
    int *at = new (std::nothrow) int[count + 1];
    if (!at) return D1_E_ARG;
    const MuonWork w = muon_work(t, count, h, at, muon_order(t, count, h, at));
    delete[] at;
    return w.total;
}

int d1_muon_check(const D1Muon *h) { return muon_args(nullptr, 0, h) && reach_of(h) < 3.8 ? 0 : D1_E_ARG; }

int d1_muon_step(const D1MuonTensor *t, int count, const D1Muon *h, int32_t *ctl, void *work, int64_t work_bytes, void *stream) {
    if (!muon_args(t, count, h) || ((uintptr_t)ctl & 3) || (h->part && !ctl)) return D1_E_ARG;
    if (d1_muon_check(h)) return D1_E_ARG;
    int *at = new (std::nothrow) int[count + 1];
    if (!at) return (int)hipErrorOutOfMemory;
    const int live = muon_order(t, count, h, at);
    const MuonWork w = muon_work(t, count, h, at, live);
    int code = D1_E_ARG;
    if (!w.total || (work && work_bytes >= w.total && !((uintptr_t)work & 255)))      // none for no matrices
        code = muon_run(t, h, ctl, (char *)work, w, at, live, (hipStream_t)stream);
    delete[] at;
    return code;
}
}
