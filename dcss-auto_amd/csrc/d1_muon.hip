// d1ops: updates orthogonalised by Newton-Schulz products, and the momentum step made of them, gfx950.
//
// X = U / (|U|_F + eps), on the side with fewer rows; then `steps` times, with (a, b, c) an odd quintic's coefficients that
// pull every singular value towards 1:
//   A = X X^T;  B = a I + b A + c A A;  X = B X
// Matrix instructions take 16-bit operands. A value is held as fp16 (one term: for results in 16 bits, 11 bits of
// mantissa where bf16 would leave 8), or as the sum of two fp16 halves (for results in 32 bits): hi = fp16(v),
// lo = fp16(v - hi), 22 bits, and a product is hi hi + hi lo + lo hi in one fp32 accumulator, three instructions for one.
// X, A and B are held 2^12 times as large, which keeps both halves of entries down to 2^-14 of the largest out of fp16's
// subnormal range; entries stay under 2^3, checked on the host from the coefficients.
//
// All operands lie in fragment order (d1_frag.h): a wave's operand of one instruction, 32 rows by 16 of the contraction, is
// one contiguous kilobyte, so loads are whole and LDS tiles are plain copies without conflicts. Rows and columns
// are padded with zeros to 64. A product P Q^T contracts adjacent elements of both: X for A; A (symmetric) for B;
// B and X^T for the new X. So X is kept in both orders and an epilogue writes its tile in both. A and B are symmetric:
// only tiles on and under the diagonal are computed, and written in both places.
#include <math.h>

#include <new>

#include "d1_rows.h"

namespace d1o {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef d1f::floatx16 acc_t;
typedef d1f::u32x4 u32x4;

constexpr int GROUP = 32;                  // matrices of a launch
constexpr int NORM_PARTS = 256;            // workgroups that sum a matrix's squares
constexpr float SCALE = 4096.f;            // of X, A and B as they are held
enum { GRAM, POLY, APPLY, LAST };
enum { C_STEP, C_SKIPPED, C_GO = 6 };

// a matrix as the products see it: m <= n after the turn, M and N their multiples of 64
struct Mat {
    _Float16 *x, *xt[2], *a, *b;           // planes of halves follow each other: hi, then lo
    void *out, *copy;                      // rows x cols as the caller has them
    float size, keep;                      // of a step: out = out * keep - size * O, else out = O
    int32_t rows, cols, m64, n64;
    int32_t last_tile;                     // tiles of this and all matrices before, for the launch
    uint8_t flip, type, step, pad;
};
struct Mats {
    Mat t[GROUP];
    const int32_t *ctl;
    float ca, cb, cc;
    int32_t count, turn, mode;             // turn: which xt is current
};
// and as its elements come and go
struct Source {
    const void *g;                         // the gradient, or the matrix itself
    float *mom;                            // null: the matrix itself
    _Float16 *x, *xt;
    int32_t rows, cols, m64, n64, last_tile, parts;
    uint8_t flip, type, pad[2];
};
struct Sources {
    Source t[GROUP];
    double *sums;                          // [matrix][NORM_PARTS], of the group's first
    double *scales;
    int32_t *parts;                        // how many sums each matrix has
    const int32_t *ctl;
    float mu;
    int32_t count, nesterov;
};

template <class T>
__device__ __forceinline__ int find(const T *t, int count, int i, int &within) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (i < t[mid].last_tile)
            hi = mid;
        else
            lo = mid + 1;
    }
    within = i - (lo ? t[lo - 1].last_tile : 0);
    return lo;
}

__device__ __forceinline__ float element(const void *p, int type, int64_t i) {
    return type == D1_FP32 ? ((const float *)p)[i] : type == D1_BF16 ? (float)((const __bf16 *)p)[i] : (float)((const _Float16 *)p)[i];
}
// what is orthogonalised, and the new momentum
__device__ __forceinline__ float update_of(const Source &t, const Sources &s, int64_t i, float &m) {
    const float g = element(t.g, t.type, i);
    if (!t.mom) return g;
    m = s.mu * t.mom[i] + g;
    return s.nesterov ? __builtin_fmaf(s.mu, m, g) : m;
}

// sums of squares, a share of the matrix a workgroup
__global__ __launch_bounds__(256) void k_muon_norm(const Sources s) {
    __shared__ double sh[4];
    int part;
    const int k = find(s.t, s.count, blockIdx.x, part);
    const Source &t = s.t[k];
    const int64_t n = (int64_t)t.rows * t.cols;
    double sum = 0.0;
    for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < n; i += (int64_t)t.parts * 256) {
        float m;
        const double u = update_of(t, s, i, m);
        sum = __builtin_fma(u, u, sum);
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
        for (int i = threadIdx.x & 63; i < parts[k]; i += 64) sum += sums[k * NORM_PARTS + i];
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
    __shared__ float tile[64][65];
    if (s.ctl && !s.ctl[C_GO]) return;
    int within;
    const int k = find(s.t, s.count, blockIdx.x, within);
    const Source &t = s.t[k];
    const double scale = s.scales[k];
    const int cols64 = t.flip ? t.m64 : t.n64;
    const int r0 = within / cols64 * 64, c0 = within % cols64 * 64;
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int r = r0 + (e >> 6), c = c0 + (e & 63);
        float v = 0.f;
        if (r < t.rows && c < t.cols) {
            const int64_t i = (int64_t)r * t.cols + c;
            float m;
            const float u = update_of(t, s, i, m);
            if (t.mom) t.mom[i] = m;
            v = (float)((double)u * scale);
        }
        tile[e >> 6][e & 63] = v;
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
    bool both;                // off the diagonal of a symmetric result: written in both places
};

// the launch's tile `i` of TILE x TILE
template <int TILE>
__device__ __forceinline__ int job_of(const Mats &s, int i, Job &job) {
    int within;
    const int k = find(s.t, s.count, i, within);
    const Mat &t = s.t[k];
    const int64_t pm = plane_of(t.m64, t.m64), px = plane_of(t.m64, t.n64);
    job.both = false;
    if (s.mode == GRAM || s.mode == POLY) {
        job.p = s.mode == GRAM ? Operand{t.x, px, t.m64 * 2, t.n64 * 4} : Operand{t.a, pm, t.m64 * 2, t.m64 * 4};
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
        if (s.mode == LAST && t.flip) {
            const Operand o = job.p;
            job.p = job.q;
            job.q = o;
        }
        const int down = (job.p.rb * 32 + TILE - 1) / TILE;
        job.bi = within % down;
        job.bj = within / down;
    }
    return k;
}

__device__ __forceinline__ acc_t mma(half8 a, half8 b, acc_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// A 32 x 32 result: lane l of register r holds row 8 (r / 4) + 4 (l / 32) + r % 4 of block I, column l % 32 of block J.
// `scratch`: the wave's 32 x 40 halves of LDS.
template <int TERMS>
__device__ __forceinline__ void put_tile(const Mats &s, const Mat &t, const Job &job, acc_t d, int I, int J, _Float16 *scratch) {
    const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
    if (I >= job.p.rb || J >= job.q.rb) return;              // the whole wave
    if (s.mode == LAST) {
        const int c = J * 32 + col;
        const float scale = 1.f / (SCALE * SCALE);
        if (c >= t.cols) return;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int row = I * 32 + d1f::drow(r, h);
            if (row >= t.rows) continue;
            const int64_t i = (int64_t)row * t.cols + c;
            float v = d[r] * scale;
            if (t.step) v = element(t.out, t.type, i) * t.keep - t.size * v;
            if (t.type == D1_FP32) ((float *)t.out)[i] = v;
            else if (t.type == D1_BF16) ((__bf16 *)t.out)[i] = (__bf16)v;
            else ((_Float16 *)t.out)[i] = (_Float16)v;
            if (t.copy) ((__bf16 *)t.copy)[i] = (__bf16)v;
        }
        return;
    }
    _Float16 *to = s.mode == GRAM ? t.a : s.mode == POLY ? t.b : t.xt[s.turn ^ 1];      // rows J, contraction I
    const int nch = t.m64;
    const int64_t plane = s.mode == APPLY ? plane_of(t.m64, t.n64) : plane_of(t.m64, t.m64);
    const int64_t at = ((((int64_t)J * nch + (I >> 1)) * 4) * 64 + col + 32 * (I & 1)) * 8 + 4 * h;
    half4 hi[4], lo[4];
#pragma unroll
    for (int g = 0; g < 4; g++) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = d[4 * g + j] * (1.f / SCALE);
        if (s.mode == POLY) {
            const half4 ah = *(const half4 *)(t.a + at + g * 512);
            half4 al = {0, 0, 0, 0};
            if (TERMS == 3) al = *(const half4 *)(t.a + plane + at + g * 512);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float a = TERMS == 3 ? (float)ah[j] + (float)al[j] : (float)ah[j];
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
    if (s.mode != APPLY && !job.both) return;
    // the other order: rows I, contraction J
    if (s.mode == APPLY) to = t.x;
    const int nch2 = s.mode == APPLY ? t.n64 : t.m64;
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

// Small results: a workgroup a tile of 32 SIDE, its waves share the contraction and join in LDS; operands straight from
// the caches into registers.
template <int TERMS, int SIDE>
__global__ __launch_bounds__(256) void k_muon_small(const Mats s) {
    constexpr int W = 4, PL = TERMS == 3 ? 2 : 1;
    __shared__ float sums[W][SIDE * SIDE][16][64];
    __shared__ __attribute__((aligned(16))) _Float16 scratch[W][32 * 40];
    if (s.ctl && !s.ctl[C_GO]) return;
    Job job;
    const Mat &t = s.t[job_of<32 * SIDE>(s, blockIdx.x, job)];
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
    const int chunks = job.p.k16 / 4, per = (chunks + W - 1) / W;
    const int lo = wave * per, hi = lo + per < chunks ? lo + per : chunks;
    for (int c = lo; c < hi; c++) {
        half8 a[4][PL][SIDE], b[4][PL][SIDE];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int pl = 0; pl < PL; pl++)
#pragma unroll
                for (int i = 0; i < SIDE; i++) {
                    a[k][pl][i] = *(const half8 *)(p[i] + pl * job.p.plane + (c * 4 + k) * 512);
                    b[k][pl][i] = *(const half8 *)(q[i] + pl * job.q.plane + (c * 4 + k) * 512);
                }
#pragma unroll
        for (int k = 0; k < 4; k++)
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
    for (int e = wave; e < SIDE * SIDE; e += W) {
        acc_t d;
#pragma unroll
        for (int r = 0; r < 16; r++) d[r] = (sums[0][e][r][lane] + sums[1][e][r][lane]) + (sums[2][e][r][lane] + sums[3][e][r][lane]);
        put_tile<TERMS>(s, t, job, d, job.bi * SIDE + e / SIDE, job.bj * SIDE + e % SIDE, scratch[wave]);
    }
}

// Large results: a workgroup a tile of TILE x TILE, operands through two LDS buffers: while one is multiplied the next
// stage lands in the other, straight from memory.
constexpr int waves_of(int tile) { return tile == 256 ? 8 : 4; }
template <int TERMS, int TILE>
struct Large {
    static constexpr int WAVES = waves_of(TILE);
    static constexpr int DOWN = 2, ACROSS = WAVES / 2;                    // waves
    static constexpr int NI = TILE / 32 / DOWN, NJ = TILE / 32 / ACROSS;  // results a wave
    static constexpr int PL = TERMS == 3 ? 2 : 1, RB = TILE / 32;
    static constexpr int QS = TERMS == 3 ? 2 : 4;                         // steps of 16 a stage
    static constexpr int PIECES = 2 * PL * RB * QS;                       // kilobytes a stage
    static constexpr int STAGE = PIECES * 512;                            // halves
};
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

template <int TERMS, int TILE>
__global__ __launch_bounds__(64 * waves_of(TILE)) void k_muon_large(const Mats s) {
    typedef Large<TERMS, TILE> L;
    __shared__ __attribute__((aligned(16))) _Float16 lds[2][L::STAGE];
    if (s.ctl && !s.ctl[C_GO]) return;
    Job job;
    const Mat &t = s.t[job_of<TILE>(s, blockIdx.x, job)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wi = wave / L::ACROSS, wj = wave % L::ACROSS;
    acc_t acc[L::NI][L::NJ];
#pragma unroll
    for (int i = 0; i < L::NI; i++)
#pragma unroll
        for (int j = 0; j < L::NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
    // kilobyte e of a stage: operand, plane, row block, step
    constexpr int MINE = L::PIECES / L::WAVES;
    const _Float16 *from[MINE];
#pragma unroll
    for (int e = 0; e < MINE; e++) {
        const int piece = e * L::WAVES + wave, k = piece % L::QS, rb = piece / L::QS % L::RB, pl = piece / (L::QS * L::RB) % L::PL,
                  side = piece / (L::QS * L::RB * L::PL);
        const Operand &o = side ? job.q : job.p;
        int R = (side ? job.bj : job.bi) * L::RB + rb;
        if (R >= o.rb) R = o.rb - 1;
        from[e] = o.p + pl * o.plane + ((int64_t)R * o.k16 + k) * 512 + lane * 8;
    }
    auto fetch = [&](int stage, int buf) {
#pragma unroll
        for (int e = 0; e < MINE; e++)
            __builtin_amdgcn_global_load_lds((global_void *)(from[e] + (int64_t)stage * L::QS * 512),
                                             (lds_void *)(lds[buf] + (e * L::WAVES + wave) * 512), 16, 0, 0);
    };
    const int stages = job.p.k16 / L::QS;
    fetch(0, 0);
    for (int st = 0; st < stages; st++) {
        __syncthreads();                   // this stage has landed, and no wave still reads the other buffer
        if (st + 1 < stages) fetch(st + 1, (st + 1) & 1);
        const _Float16 *a0 = lds[st & 1] + (wi * L::NI * L::QS) * 512 + lane * 8;
        const _Float16 *b0 = lds[st & 1] + (L::PL * L::RB * L::QS + wj * L::NJ * L::QS) * 512 + lane * 8;
#pragma unroll
        for (int k = 0; k < L::QS; k++) {
            half8 a[L::PL][L::NI], b[L::PL][L::NJ];
#pragma unroll
            for (int pl = 0; pl < L::PL; pl++) {
#pragma unroll
                for (int i = 0; i < L::NI; i++) a[pl][i] = *(const half8 *)(a0 + ((pl * L::RB + i) * L::QS + k) * 512);
#pragma unroll
                for (int j = 0; j < L::NJ; j++) b[pl][j] = *(const half8 *)(b0 + ((pl * L::RB + j) * L::QS + k) * 512);
            }
#pragma unroll
            for (int i = 0; i < L::NI; i++)
#pragma unroll
                for (int j = 0; j < L::NJ; j++) {
                    acc[i][j] = mma(a[0][i], b[0][j], acc[i][j]);
                    if (TERMS == 3) {
                        acc[i][j] = mma(a[0][i], b[L::PL - 1][j], acc[i][j]);
                        acc[i][j] = mma(a[L::PL - 1][i], b[0][j], acc[i][j]);
                    }
                }
        }
    }
    __syncthreads();                       // the buffers become the waves' scratch
    _Float16 *scratch = lds[0] + wave * 32 * 40;
#pragma unroll
    for (int i = 0; i < L::NI; i++)
#pragma unroll
        for (int j = 0; j < L::NJ; j++)
            put_tile<TERMS>(s, t, job, acc[i][j], job.bi * L::RB + wi * L::NI + i, job.bj * L::RB + wj * L::NJ + j, scratch);
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
// Kinds of kernels: 0 small tiles of 32, 1 of 64, 2 large tiles of 128, 3 of 256
constexpr int side_of(int kind) { return kind == 0 ? 32 : kind == 1 ? 64 : kind == 2 ? 128 : 256; }
inline int64_t tiles_of(int mode, const Shape &h, int side) {
    const int64_t m = ((int64_t)h.m64 * 64 + side - 1) / side, n = ((int64_t)h.n64 * 64 + side - 1) / side;
    return mode == GRAM || mode == POLY ? m * (m + 1) / 2 : m * n;
}
inline int terms_of(const D1MuonTensor &t, const D1Muon *h) { return h->terms ? h->terms : t.type == D1_FP32 ? 3 : 1; }
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
inline int kind_of(int64_t tiles256, int64_t tiles128, int64_t tiles64) {
    return tiles256 >= 192 ? 3 : tiles128 >= 192 ? 2 : tiles64 >= 192 ? 1 : 0;
}

// The singular values of X lie in [0, 1] after the norm; the largest that the steps make of them, from a fine grid and the
// slope's bound between its points. What is held has to stay under 2^3 times the scale, and below that in A = s^2.
static double reach_of(const D1Muon *h) {
    double top = 1.0;
    for (int k = 0; k < h->steps; k++) {
        double most = 0.0;
        for (int i = 0; i <= 4096; i++) {
            const double x = top * i / 4096, x2 = x * x, b = h->a + h->b * x2 + h->c * x2 * x2;
            if (!(fabs(b) < 15.0) || !(x2 < 15.0)) return INFINITY;
            if (fabs(b * x) > most) most = fabs(b * x);
        }
        top = most * 1.001 + 1e-3;
        if (!(top < 3.8)) return INFINITY;
    }
    return top;
}

static bool muon_args(const D1MuonTensor *t, int count, const D1Muon *h) {
    if (count < 0 || (count && !t) || !h || (h->terms != 0 && h->terms != 1 && h->terms != 3)) return false;
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

struct MuonWork {
    int64_t parts, sums, scales, mats;    // offsets; the rest is one group's operands
};
static int64_t muon_work(const D1MuonTensor *t, int count, const D1Muon *h, MuonWork &w) {
    w.parts = 0;
    w.sums = ((int64_t)count * 4 + 255) & ~(int64_t)255;
    w.scales = w.sums + (int64_t)count * NORM_PARTS * 8;
    w.mats = (w.scales + (int64_t)count * 8 + 255) & ~(int64_t)255;
    int64_t most = 0, bytes = 0;
    for (int i = 0; i < count; i++) {
        const int64_t b = t[i].rows && t[i].cols ? mat_bytes(t[i], terms_of(t[i], h)) : 0;
        most = b > most ? b : most;
        bytes += b;
    }
    // a group is at most GROUP_BYTES or one matrix
    const int64_t room = bytes < GROUP_BYTES ? bytes : GROUP_BYTES > most ? GROUP_BYTES : most;
    return w.mats + room;
}

template <int TERMS>
static void muon_products(const Mats &s, int64_t tiles, int kind, hipStream_t stream) {
    const dim3 grid((unsigned)tiles);
    if (kind == 3)
        hipLaunchKernelGGL((k_muon_large<TERMS, 256>), grid, dim3(512), 0, stream, s);
    else if (kind == 2)
        hipLaunchKernelGGL((k_muon_large<TERMS, 128>), grid, dim3(256), 0, stream, s);
    else if (kind == 1)
        hipLaunchKernelGGL((k_muon_small<TERMS, 2>), grid, dim3(256), 0, stream, s);
    else
        hipLaunchKernelGGL((k_muon_small<TERMS, 1>), grid, dim3(256), 0, stream, s);
}

static int muon_run(const D1MuonTensor *t, int count, const D1Muon *h, int32_t *ctl, char *work, const MuonWork &w, hipStream_t stream) {
    int *at = new (std::nothrow) int[count + 1];
    if (!at) return (int)hipErrorOutOfMemory;
    int live = 0;
    for (int terms : {3, 1})
        for (int i = 0; i < count; i++)
            if (t[i].rows && t[i].cols && terms_of(t[i], h) == terms) at[live++] = i;
    double *sums = (double *)(work + w.sums), *scales = (double *)(work + w.scales);
    int32_t *parts = (int32_t *)(work + w.parts);
    auto sources = [&](int from, int to, bool prepare, Sources &s) {
        s = Sources{};
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
            o.last_tile = (int32_t)tiles;
        }
        return tiles;
    };
    for (int from = 0; from < live;) {
        const int to = live - from < GROUP ? live : from + GROUP;
        Sources s;
        const int64_t tiles = sources(from, to, false, s);
        hipLaunchKernelGGL(k_muon_norm, dim3((unsigned)tiles), dim3(256), 0, stream, s);
        from = to;
    }
    hipLaunchKernelGGL(k_muon_begin, dim3(1), dim3(1024), 0, stream, sums, scales, parts, live, h->eps, ctl);
    for (int from = 0; from < live;) {
        const int to = group_end(t, at, live, from, h), terms = terms_of(t[at[from]], h);
        Sources s;
        const int64_t tiles = sources(from, to, true, s);
        Mats p{};
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
        for (int step = 0; step < h->steps; step++) {
            p.turn = step & 1;
            for (int mode : {(int)GRAM, (int)POLY, step + 1 < h->steps ? (int)APPLY : (int)LAST}) {
                p.mode = mode;
                int64_t n[4] = {};
                for (int k = 0; k < p.count; k++)
                    for (int kind = 0; kind < 4; kind++) n[kind] += tiles_of(mode, shape_of(t[at[from + k]]), side_of(kind));
                const int kind = kind_of(n[3], n[2], n[1]);
                int64_t sum = 0;
                for (int k = 0; k < p.count; k++) {
                    sum += tiles_of(mode, shape_of(t[at[from + k]]), side_of(kind));
                    p.t[k].last_tile = (int32_t)sum;
                }
                if (terms == 3)
                    muon_products<3>(p, sum, kind, stream);
                else
                    muon_products<1>(p, sum, kind, stream);
            }
        }
        from = to;
    }
    delete[] at;
    return (int)hipGetLastError();
}

}  // namespace d1o

using namespace d1o;

extern "C" {
int64_t d1_muon_work_bytes(const D1MuonTensor *t, int count, const D1Muon *h) {
    if (!muon_args(t, count, h)) return D1_E_ARG;
    MuonWork w;
    return muon_work(t, count, h, w);
}

int d1_muon_check(const D1Muon *h) { return muon_args(nullptr, 0, h) && reach_of(h) < 3.8 ? 0 : D1_E_ARG; }

int d1_muon_step(const D1MuonTensor *t, int count, const D1Muon *h, int32_t *ctl, void *work, int64_t work_bytes, void *stream) {
    if (!muon_args(t, count, h) || ((uintptr_t)ctl & 3)) return D1_E_ARG;
    if (d1_muon_check(h)) return D1_E_ARG;
    MuonWork w;
    const int64_t need = muon_work(t, count, h, w);
    if (!work || work_bytes < need || ((uintptr_t)work & 255)) return D1_E_ARG;
    return muon_run(t, count, h, ctl, (char *)work, w, (hipStream_t)stream);
}
}
