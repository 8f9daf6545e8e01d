// d1ops: log probabilities of given tokens with entropy, top alternatives and gradient, gfx950.
//
// Of a row's allowed entries x with maximum m:  S = sum e^(x-m),  E = sum e^(x-m) (x-m), then
//   logp = (x[t] - m) - log S,   entropy = log S - E/S  (both terms are sums of one sign: no
//   cancellation for a row that is sure of one entry),   p = e^(x-m) / S,
//   dx = g (1[t] - p) - h p (log p + entropy)  with g, h the gradients of logp and entropy.
// Each entry is read once: m, S and E run along, rescaled when m grows. The backward pass reads m
// and S again and no sums.
//
// Rows of up to 512 entries stay in the registers of 4 to 32 lanes (k_tokens_small). A longer row
// is cut into segments of one workgroup each, as many as fill the card when rows are few
// (k_tokens_part), and where there are several k_tokens_join adds their m, S, E and merges their best entries.
//
// Alternatives are ordered by a 64-bit key: the value's order-preserving bits, then the
// complemented index, so keys are distinct and the lowest index wins among equal values.
#include "d1_rows.h"

namespace d1o {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float FAR = -1e4f;          // below any difference whose exponential is not 0
constexpr int SMALL_VOCAB = 512, SMALL_BWD_VOCAB = 1024;

// e^d by the hardware's 2^x. Its argument d log2(e) is rounded once, which leaves the result a relative error of up to 1.5 |d| u
// (u = 2^-24: 4e-6 for an entry at d = -40, which is e^-40 of the largest). In the sums an entry weighs e^d, and |d| e^d is
// 0.37 at most, so they stay within half a u of it; only the gradient of an entry far below the largest carries the error whole, 4e-6
// of a number that is 4e-18 of the row's. An argument in two words would need the exponential's fraction and power apart.
__device__ __forceinline__ float exp_nat(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
// e (x-m) for e = exp(x-m): 0 also for x = -inf, NaN where e is
__device__ __forceinline__ float weighted(float e, float d) { return e * fmaxf(d, FAR); }

// order-preserving bits: larger value, larger word; -0 as +0, NaN above +inf. No value maps to 0,
// which stands for none, or to ~0, which is above all.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0xFFFFFFFEu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);   // NaN's word gives a NaN
}
__device__ __forceinline__ uint64_t key_of(float x, int index) { return ((uint64_t)ordered(x) << 32) | (uint32_t)~index; }
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }


// running maximum, sum of exponentials and of exponentials times differences
struct Sums {
    float m, s, e;
};
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.f : m; }
// a and b over the same base; a part without entries above -inf has s = e = 0
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m), base = finite_base(m);
    const float da = a.m - base, db = b.m - base;
    const float ca = exp_nat(da), cb = exp_nat(db);
    // s and e of a part are about its own maximum: x - m = (x - a.m) + (a.m - m)
    return {m, ca * a.s + cb * b.s, ca * __builtin_fmaf(a.s, fmaxf(da, FAR), a.e) + cb * __builtin_fmaf(b.s, fmaxf(db, FAR), b.e)};
}
template <int LANES>
__device__ __forceinline__ Sums lanes_joined(Sums a) {
    const float m = lanes_max<LANES>(a.m), d = a.m - finite_base(m), c = exp_nat(d);
    return {m, lanes_sum<LANES>(c * a.s), lanes_sum<LANES>(c * __builtin_fmaf(a.s, fmaxf(d, FAR), a.e))};
}

struct Args {
    const void *logits;
    int64_t rows, stride;
    int vocab, top;
    const int64_t *tokens;
    const uint8_t *mask;
    int64_t mask_stride;
    float *logp, *entropy, *stats;
    int64_t *top_ids;
    float *top_logp;
};

// logp of a token whose entry is x (x is -inf where it is masked)
__device__ __forceinline__ float logp_of(float x, Sums t, float base, float ls) {
    return t.s == 0.f ? -INFINITY : (x - base) - ls;
}
// logp of what is no token: padding, or an index past the row
__device__ __forceinline__ float logp_of_none(int64_t tok) { return tok < 0 ? 0.f : __builtin_nanf(""); }
__device__ __forceinline__ void put_row(const Args &a, int64_t row, Sums t, float base, float ls) {
    a.entropy[row] = t.s == 0.f ? 0.f : ls - t.e / t.s;
    a.stats[2 * row] = base;
    a.stats[2 * row + 1] = t.s;
}
// A long row's token and its entry, asked for before the row is read (two loads, one after the other).
struct Given {
    int64_t tok;
    float x;
};
template <class T>
__device__ __forceinline__ Given given_of(const Args &a, int64_t row) {
    Given g = {a.tokens[row], -INFINITY};
    if (g.tok >= 0 && g.tok < a.vocab && (!a.mask || a.mask[row * a.mask_stride + g.tok]))
        g.x = (float)((const T *)a.logits)[row * a.stride + g.tok];
    return g;
}
// what one lane writes of a long row once its sums are whole
__device__ __forceinline__ void finish(const Args &a, int64_t row, Sums t, Given g) {
    const float base = finite_base(t.m), ls = logf(t.s);
    a.logp[row] = g.tok < 0 || g.tok >= a.vocab ? logp_of_none(g.tok) : logp_of(g.x, t, base, ls);
    put_row(a, row, t, base, ls);
}
__device__ __forceinline__ void put_top(const Args &a, int64_t row, int k, uint64_t key, float base, float ls, float s) {
    const bool none = (key >> 32) == 0;
    a.top_ids[row * a.top + k] = none ? -1 : index_of(key);
    a.top_logp[row * a.top + k] = none || s == 0.f ? -INFINITY : (value_of((uint32_t)(key >> 32)) - base) - ls;
}

// ---- rows of up to LANES * CH * 4 entries, one row for LANES lanes, 4 adjacent entries a chunk

template <class T, int LANES, int CH, bool MASK>
struct SmallRow {
    float x[CH][4];       // -inf where `in` is not set
    bool in[CH][4];       // an allowed entry of the lane's
    int at[CH];           // index of the chunk's first entry
    // chunks of rows of 4 entries or more are whole loads; `shared`: what they hold of the lane before counts too
    __device__ __forceinline__ void read(const T *logits, const uint8_t *mask, int vocab, int lane, bool shared) {
        Pack<T, 4> p[CH];
        Pack<uint8_t, 4> q[CH];
        int skip[CH];
        if (vocab >= 4) {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const Place w = place_of<4>((c * LANES + lane) * 4, vocab);
                at[c] = w.at;
                skip[c] = w.skip;
                p[c] = load<T, 4>(logits + w.at);
                if (MASK) q[c] = load<uint8_t, 4>(mask + w.at);
            }
        } else {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                at[c] = (c * LANES + lane) * 4;
                skip[c] = at[c] ? 4 : 0;
                p[c] = load_part<T, 4>(logits, at[c] ? 0 : vocab, (T)0.f);
                if (MASK) q[c] = load_part<uint8_t, 4>(mask, at[c] ? 0 : vocab, 0);
            }
        }
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                in[c][i] = (shared ? skip[c] < 4 : i >= skip[c]) && at[c] + i < vocab && (!MASK || q[c].v[i]);
                x[c][i] = in[c][i] ? (float)p[c].v[i] : -INFINITY;
            }
    }
};

// 256 / LANES rows a workgroup, each read once into registers; alternatives one after the other, the largest key over the
// row's lanes each time. Small calls are the launch (8,192 x 16 fp32 2.7 us); with alternatives the instructions of their
// reductions bound it (65,536 x 25 with 3 and a mask 6.5 us; 62,655 x 89 bf16 with 20 34 us, 7.7 at the bytes' rate).
template <class T, int LANES, int CH, bool MASK>
__global__ __launch_bounds__(256) void k_tokens_small(const Args a) {
    constexpr int GROUPS = 256 / LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    for (int64_t row = (int64_t)blockIdx.x * GROUPS + group; row < a.rows; row += (int64_t)gridDim.x * GROUPS) {
        SmallRow<T, LANES, CH, MASK> r;
        r.read((const T *)a.logits + row * a.stride, MASK ? a.mask + row * a.mask_stride : nullptr, a.vocab, lane, false);
        const int64_t tok = a.tokens[row];
        float m = -INFINITY;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) m = fmaxf(m, r.x[c][i]);
        m = lanes_max<LANES>(m);
        const float base = finite_base(m);
        float s = 0.f, e = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float d = r.x[c][i] - base, w = exp_nat(d);
                s += w;
                e += weighted(w, d);
            }
        s = lanes_sum<LANES>(s);
        e = lanes_sum<LANES>(e);
        const Sums t = {m, s, e};
        const float ls = logf(s);
        // the lane that holds the token's entry writes its logp: no second, dependent read of the row
        if (lane == 0) {
            put_row(a, row, t, base, ls);
            if (tok < 0 || tok >= a.vocab) a.logp[row] = logp_of_none(tok);
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int64_t col = (c * LANES + lane) * 4;
            if (tok >= col && tok < col + 4 && tok < a.vocab) {
                const int at = (int)tok - r.at[c];
                const float x = at < 2 ? (at ? r.x[c][1] : r.x[c][0]) : (at == 2 ? r.x[c][2] : r.x[c][3]);
                a.logp[row] = logp_of(x, t, base, ls);
            }
        }
        if (a.top) {
            uint32_t word[CH][4];        // 0: not an entry, or taken
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) word[c][i] = r.in[c][i] ? ordered(r.x[c][i]) : 0;
            for (int k = 0; k < a.top; k++) {
                uint32_t best = 0, first = 0xFFFFFFFFu;
#pragma unroll
                for (int c = 0; c < CH; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) best = best > word[c][i] ? best : word[c][i];
                best = lanes_u<LANES>(best, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
#pragma unroll
                for (int c = CH - 1; c >= 0; c--)
#pragma unroll
                    for (int i = 3; i >= 0; i--) first = word[c][i] == best ? r.at[c] + i : first;
                first = lanes_u<LANES>(first, [](uint32_t p, uint32_t q) { return p < q ? p : q; });
#pragma unroll
                for (int c = 0; c < CH; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) word[c][i] = (uint32_t)(r.at[c] + i) == first ? 0 : word[c][i];
                if (lane == 0) put_top(a, row, k, ((uint64_t)best << 32) | (uint32_t)~first, base, ls, s);
            }
        }
    }
}

// ---- longer rows: segments

// Vectors of 16 bytes that a thread takes at once, a round of its loop: two; four (512 x 50,001 fp16 31 us against 28, 4,096
// x 131,072 bf16 210 against 192) and eight (222) cost more waves than they hide.
constexpr int AT_ONCE = 2, KEEP = 512, ROUND = 4;

struct Parts {
    float *sums;              // [rows][splits][4]: m, s, e
    uint64_t *keys;           // [rows][splits][top]
    int part, splits, seg;    // threads of a workgroup, segments a row, entries of one (a multiple of a vector)
};

// VEC allowed entries of a segment from `at` on; the first `skip` and what the mask leaves out read -inf
template <class T, int VEC, bool MASK>
__device__ __forceinline__ void read_vec(const T *x, const uint8_t *mask, Place w, Pack<T, VEC> &p, Pack<uint8_t, VEC> &q) {
    p = load<T, VEC>(x + w.at);
    if (MASK) q = load<uint8_t, VEC>(mask + w.at);
}
template <class T, int VEC, bool MASK>
__device__ __forceinline__ void widen_vec(const Pack<T, VEC> &p, const Pack<uint8_t, VEC> &q, int skip, float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = j >= skip && (!MASK || q.v[j]) ? (float)p.v[j] : -INFINITY;
}

// what the lanes of a wave wrote to LDS is there for the others after this
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int PART>
__device__ __forceinline__ void block_sync() {
    if (PART == 64)
        wave_sync();
    else
        __syncthreads();
}

// a bound on the k-th largest of the lanes' words (N a lane) from below, exact in its first 18 bits: bit by bit from the top,
// as long as k words stay at or above it
template <int N>
__device__ __forceinline__ uint32_t kth_word(const uint32_t (&word)[N], int k) {
    uint32_t floor = 0;
#pragma unroll
    for (int bit = 31; bit >= 14; bit--) {
        const uint32_t at = floor | (1u << bit);
        int above = 0;
#pragma unroll
        for (int i = 0; i < N; i++) above += __popcll(__ballot(word[i] >= at));
        if (above >= k) floor = at;
    }
    return floor;
}

// A wave's list of keys in LDS: takes keys in any order, keeps at least the `top` largest seen.
struct TopList {
    uint64_t *list, *sorted;     // KEEP and D1_TOKENS_MAX_TOP keys
    int top, count;
    uint64_t below;              // keys up to this one are not among the largest

    // leaves out keys whose word is below the top-th largest word's first bits: where few are equal, little
    // more than `top` stay (a list of 242 keys was sorted in 10 us without)
    __device__ __forceinline__ void prune(int lane) {
        uint64_t key[KEEP / 64];
        uint32_t word[KEEP / 64];
        wave_sync();
#pragma unroll
        for (int i = 0; i < KEEP / 64; i++) {
            key[i] = i * 64 + lane < count ? list[i * 64 + lane] : 0;
            word[i] = (uint32_t)(key[i] >> 32);
        }
        const uint32_t floor = kth_word<KEEP / 64>(word, top);
        wave_sync();
        count = 0;
#pragma unroll
        for (int i = 0; i < KEEP / 64; i++) {
            const uint64_t stay = __ballot(word[i] && word[i] >= floor);
            if (word[i] && word[i] >= floor) list[count + __popcll(stay & ((1ull << lane) - 1))] = key[i];
            count += __popcll(stay);
        }
    }
    // the `top` largest to `sorted`, falling; places without a key are 0. A key's place is the number of larger ones.
    __device__ __forceinline__ void sort(int lane) {
        if (count > 64) prune(lane);
        wave_sync();
        if (lane < top) sorted[lane] = 0;
        wave_sync();
        for (int i0 = 0; i0 < count; i0 += 64) {
            const uint64_t mine = i0 + lane < count ? list[i0 + lane] : 0;
            int larger = 0;
            for (int j0 = 0; j0 < count; j0 += 8) {
                uint64_t key[8];
#pragma unroll
                for (int j = 0; j < 8; j++) key[j] = list[j0 + j];     // KEEP is a multiple of 8
#pragma unroll
                for (int j = 0; j < 8; j++) larger += j0 + j < count && key[j] > mine;
            }
            if (mine && larger < top) sorted[larger] = mine;
        }
        wave_sync();
    }
    __device__ __forceinline__ void shrink(int lane) {
        sort(lane);
        if (lane < top) list[lane] = sorted[lane];
        below = sorted[top - 1];
        count = count < top ? count : top;
        wave_sync();
    }
    // ROUND keys a lane (0: none); the whole wave calls
    __device__ __forceinline__ void add(const uint64_t (&key)[ROUND], int lane) {
#pragma unroll
        for (int u = 0; u < ROUND; u++) {
            const uint64_t take = __ballot(key[u] > below);
            if (key[u] > below) list[count + __popcll(take & ((1ull << lane) - 1))] = key[u];
            count += __popcll(take);
        }
        if (count > KEEP - 64 * ROUND) shrink(lane);
    }
};

// A segment of a row on PART threads: m, S, E in one pass; for alternatives each lane also keeps its largest value, and the
// `top`-th largest of those bounds what a second look at the segment (from the caches) collects: only lanes whose largest
// passes the bound look again. Without alternatives bound by memory (4,096 x 131,072 bf16 190 us, 5.6 TB/s), with them by
// the collecting and sorting of one workgroup (1 x 131,072 with 20 10.4 us in all).
template <class T, int PART, bool MASK, bool TOP>
__global__ __launch_bounds__(PART) void k_tokens_part(const Args a, const Parts parts) {
    constexpr int VEC = 16 / (int)sizeof(T), STEP = PART * VEC, WAVES = PART / 64;
    __shared__ Sums wave_sums[WAVES];
    __shared__ uint32_t words[TOP ? PART : 1];
    __shared__ int wave_count[WAVES];
    __shared__ uint8_t lanes_of[WAVES][64];
    __shared__ uint64_t found[TOP ? WAVES : 1][TOP ? KEEP : 1], sorted[TOP ? WAVES : 1][TOP ? D1_TOKENS_MAX_TOP : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t units = a.rows * parts.splits;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t row = unit / parts.splits;
        const int split = (int)(unit - row * parts.splits), begin = split * parts.seg;
        const int n = a.vocab - begin < parts.seg ? a.vocab - begin : parts.seg;
        const T *x = (const T *)a.logits + row * a.stride + begin;
        const uint8_t *mask = MASK ? a.mask + row * a.mask_stride + begin : nullptr;
        Sums t = {-INFINITY, 0.f, 0.f};
        Given given = {-1, 0.f};
        if (parts.splits == 1 && threadIdx.x == 0) given = given_of<T>(a, row);
        uint64_t allowed = 0;            // of TOP and MASK: not 0 where the lane saw an allowed entry (or one of its neighbour's)
        auto take = [&](int i, bool whole) {       // AT_ONCE vectors from entry i on, every lane of a whole round inside the row
            Pack<T, VEC> p[AT_ONCE];
            Pack<uint8_t, VEC> q[AT_ONCE];
            Place w[AT_ONCE];
            float v[AT_ONCE][VEC];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                w[u] = whole ? Place{i + u * STEP, 0} : place_of<VEC>(i + u * STEP, n);
                read_vec<T, VEC, MASK>(x, mask, w[u], p[u], q[u]);
            }
            if (TOP && MASK) {
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) {
                    uint64_t bits = 0;
                    __builtin_memcpy(&bits, &q[u], sizeof q[u]);
                    allowed |= bits;
                }
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) widen_vec<T, VEC, MASK>(p[u], q[u], w[u].skip, v[u]);
            float m = t.m;
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
                for (int j = 0; j < VEC; j++) m = fmaxf(m, v[u][j]);
            const float base = finite_base(m), d0 = t.m - base, c = exp_nat(d0);
            t.e = c * __builtin_fmaf(t.s, fmaxf(d0, FAR), t.e);
            t.s = c * t.s;
            t.m = m;
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float d = v[u][j] - base, e = exp_nat(d);
                    t.s += e;
                    t.e += weighted(e, d);
                }
        };
        int i0 = 0;
        for (; i0 + STEP * AT_ONCE <= n; i0 += STEP * AT_ONCE) take(i0 + threadIdx.x * VEC, true);
        if (i0 < n) take(i0 + threadIdx.x * VEC, false);
        const Sums wave_sum = lanes_joined<64>(t);
        uint32_t most = 0;               // of TOP: a word that no entry of the lane passes
        if (TOP) {
            // The maximum leaves NaN out, which is the largest of all; the sum knows of it (or of +inf).
            // A lane without an entry above -inf may still hold allowed ones there: it counts as one, unless its mask
            // allows none (8 x 27,868, one of them masked out: 12 us, 25 where that one is looked through whole).
            const bool odd = t.s != t.s;
            const uint32_t word = (int)threadIdx.x * VEC >= n || (MASK && !allowed) ? 0 : odd && t.m != INFINITY ? 0xFFFFFFFEu : ordered(t.m);
            words[threadIdx.x] = word;
            most = odd ? 0xFFFFFFFEu : word;
        }
        if (lane == 0) wave_sums[wave] = wave_sum;
        block_sync<PART>();
        Sums all = wave_sums[0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) all = joined(all, wave_sums[w]);
        if (threadIdx.x == 0) {
            if (parts.splits == 1) {
                finish(a, row, all, given);
            } else {
                float *o = parts.sums + unit * 4;
                o[0] = all.m;
                o[1] = all.s;
                o[2] = all.e;
            }
        }
        if (TOP) {
            // At least `top` lanes hold an entry of this word or more, so the segment's best are no smaller;
            // only lanes that hold such an entry are looked through again, by their whole wave.
            uint32_t word[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; w++) word[w] = words[w * 64 + lane];
            const uint32_t floor = kth_word<WAVES>(word, a.top);
            TopList best = {found[wave], sorted[wave], a.top, 0, 0};
            const int each = ((n + STEP - 1) / STEP) * VEC;      // entries of a lane
            const bool mine = most && most >= floor;
            const uint64_t open = __ballot(mine);
            uint8_t *who = lanes_of[wave];                       // the lanes to look through, in order
            if (mine) who[__popcll(open & ((1ull << lane) - 1))] = (uint8_t)lane;
            wave_sync();
            const int total = __popcll(open) * each;
            for (int q0 = 0; q0 < total; q0 += ROUND * 64) {
                T entry[ROUND];
                bool in[ROUND];
                int at[ROUND];
#pragma unroll
                for (int u = 0; u < ROUND; u++) {                // all loads in flight
                    const int q = q0 + u * 64 + lane, k = q / each, r = q - k * each;
                    at[u] = q < total ? (r / VEC * PART + wave * 64 + who[k]) * VEC + r % VEC : n;
                    in[u] = at[u] < n;
                    entry[u] = in[u] ? x[at[u]] : (T)0.f;
                    if (MASK) in[u] = in[u] && mask[at[u]];
                }
                uint64_t key[ROUND];
#pragma unroll
                for (int u = 0; u < ROUND; u++) {
                    key[u] = in[u] ? key_of((float)entry[u], begin + at[u]) : 0;
                    if ((uint32_t)(key[u] >> 32) < floor) key[u] = 0;
                }
                best.add(key, lane);
            }
            if (WAVES > 1) {
                if (best.count > 64) best.shrink(lane);
                if (lane == 0) wave_count[wave] = best.count;
                block_sync<PART>();
            }
            if (wave == 0) {       // the waves' lists, 64 keys each at most
#pragma unroll
                for (int w0 = 1; w0 < WAVES; w0 += ROUND) {
                    uint64_t key[ROUND];
#pragma unroll
                    for (int u = 0; u < ROUND; u++) key[u] = w0 + u < WAVES && lane < wave_count[w0 + u] ? found[w0 + u][lane] : 0;
                    best.add(key, lane);
                }
                best.sort(lane);
                if (parts.splits == 1) {
                    if (lane < a.top) put_top(a, row, lane, sorted[0][lane], finite_base(all.m), logf(all.s), all.s);
                } else if (lane < a.top) {
                    parts.keys[unit * a.top + lane] = sorted[0][lane];
                }
            }
        }
        block_sync<PART>();
    }
}

// one wave a row: lane l holds segment l (at most 64 segments) and walks its sorted list
template <class T>
__global__ __launch_bounds__(64) void k_tokens_join(const Args a, const Parts parts) {
    __shared__ uint64_t found[KEEP], sorted[D1_TOKENS_MAX_TOP];
    const int lane = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Sums t = {-INFINITY, 0.f, 0.f};
        const bool mine = lane < parts.splits;
        if (mine) {
            const float *p = parts.sums + (row * parts.splits + lane) * 4;
            t = {p[0], p[1], p[2]};
        }
        const uint64_t *all = parts.keys + row * parts.splits * a.top, *keys = all + lane * a.top;
        const int total = parts.splits * a.top;
        const bool flat = total <= ROUND * 64;
        constexpr int FIRST = 2 * ROUND;
        uint64_t key[FIRST];             // few keys: all of them, whoever's; many: the first of the lane's list
#pragma unroll
        for (int j = 0; j < FIRST; j++) {
            const int at = j * 64 + lane;
            key[j] = flat ? at < total ? all[at] : 0 : mine && j < a.top ? keys[j] : 0;
        }
        const Given given = given_of<T>(a, row);
        t = lanes_joined<64>(t);
        if (lane == 0) finish(a, row, t, given);
        if (a.top) {
            // the top-th largest of what is read so far bounds the row's best from below
            uint32_t word[FIRST];
#pragma unroll
            for (int j = 0; j < FIRST; j++) word[j] = (uint32_t)(key[j] >> 32);
            const uint32_t floor = kth_word<FIRST>(word, a.top);
            TopList best = {found, sorted, a.top, 0, 0};
            uint64_t four[ROUND];
            for (int k0 = 0; k0 < a.top; k0 += ROUND) {
#pragma unroll
                for (int j = 0; j < ROUND; j++) {
                    four[j] = k0 == 0 ? key[j] : k0 == ROUND ? key[ROUND + j] : mine && four[ROUND - 1] && k0 + j < a.top ? keys[k0 + j] : 0;
                    if ((uint32_t)(four[j] >> 32) < floor) four[j] = 0;
                }
                best.add(four, lane);
                if (flat || !__ballot(four[ROUND - 1] > best.below)) break;     // the lists fall: nothing larger follows
            }
            best.sort(lane);
            if (lane < a.top) put_top(a, row, lane, sorted[lane], finite_base(t.m), logf(t.s), t.s);
            wave_sync();
        }
    }
}

// ---- gradient

struct BackArgs {
    const void *logits;
    int64_t rows, stride;
    int vocab;
    const int64_t *tokens;
    const uint8_t *mask;
    int64_t mask_stride;
    const float *stats, *entropy, *dlogp, *dentropy;
    void *dlogits;
};
// dx = e^d (add + scale d) for d = x - base, and `g` more at the token. e^d is taken as the square
// of e^(d/2): the hardware's exponential has no denormal results, and p may be small where dx is not.
struct RowGrad {
    float base, add, scale, g;
    int64_t tok;
};
__device__ __forceinline__ RowGrad row_grad(const BackArgs &a, int64_t row) {
    const float s = a.stats[2 * row + 1], inv = s == 0.f ? 0.f : 1.f / s;
    RowGrad r;
    r.base = a.stats[2 * row];
    r.tok = a.tokens[row];
    const float h = a.dentropy ? a.dentropy[row] : 0.f;
    r.g = a.dlogp && r.tok >= 0 ? a.dlogp[row] : 0.f;
    if (a.dlogp && r.tok >= a.vocab) r.g = __builtin_nanf("");
    const float shift = a.dentropy && s != 0.f ? a.entropy[row] - logf(s) : 0.f;
    r.add = -inv * __builtin_fmaf(h, shift, r.g);
    r.scale = -inv * h;
    if (s == 0.f) r.add = r.scale = r.g = 0.f;
    return r;
}
__device__ __forceinline__ float grad_of(const RowGrad &r, float x) {
    const float d = x - r.base;
    const float half = __builtin_amdgcn_exp2f(d * (0.5f * LOG2E));
    return half * (half * __builtin_fmaf(r.scale, fmaxf(d, FAR), r.add));
}

// Gradients of short rows: rows on lanes as in k_tokens_small, no sums (65,536 x 25 with a mask 5.3 us, 3.4 at the bytes' rate).
template <class T, int LANES, int CH, bool MASK>
__global__ __launch_bounds__(256) void k_tokens_small_bwd(const BackArgs a) {
    constexpr int GROUPS = 256 / LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    for (int64_t row = (int64_t)blockIdx.x * GROUPS + group; row < a.rows; row += (int64_t)gridDim.x * GROUPS) {
        SmallRow<T, LANES, CH, MASK> r;
        r.read((const T *)a.logits + row * a.stride, MASK ? a.mask + row * a.mask_stride : nullptr, a.vocab, lane, true);
        const RowGrad q = row_grad(a, row);
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int col = (c * LANES + lane) * 4;
            Pack<T, 4> o;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float d = grad_of(q, r.x[c][i]) + (r.at[c] + i == q.tok ? q.g : 0.f);
                o.v[i] = (T)(r.in[c][i] ? d : 0.f);
            }
            store_part<T, 4>((T *)a.dlogits + row * a.vocab + r.at[c], col >= a.vocab ? 0 : a.vocab < 4 ? a.vocab : 4, o);
        }
    }
}

// Gradients of longer rows: an entry needs m, S and the entropy alone, so segments are independent; bound by memory (4,096 x
// 131,072 bf16 343 us at best, 6.3 TB/s of reading and writing).
template <class T, int PART, bool MASK, bool PAST>
__global__ __launch_bounds__(PART) void k_tokens_bwd(const BackArgs a, int splits, int seg) {
    constexpr int VEC = 16 / (int)sizeof(T), STEP = PART * VEC;
    const int64_t units = a.rows * splits;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t row = unit / splits;
        const int begin = (int)(unit - row * splits) * seg;
        const int n = a.vocab - begin < seg ? a.vocab - begin : seg;
        const T *x = (const T *)a.logits + row * a.stride + begin;
        const uint8_t *mask = MASK ? a.mask + row * a.mask_stride + begin : nullptr;
        T *out = (T *)a.dlogits + row * a.vocab + begin;
        const RowGrad q = row_grad(a, row);
        auto take = [&](int i, bool whole) {
            Pack<T, VEC> p[AT_ONCE];
            Pack<uint8_t, VEC> in[AT_ONCE];
            Place w[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                w[u] = whole ? Place{i + u * STEP, 0} : place_of<VEC>(i + u * STEP, n);
                read_vec<T, VEC, MASK>(x, mask, w[u], p[u], in[u]);
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float d = grad_of(q, (float)p[u].v[j]) + (begin + w[u].at + j == q.tok ? q.g : 0.f);
                    o.v[j] = (T)(!MASK || in[u].v[j] ? d : 0.f);
                }
                if (whole || w[u].skip < VEC) put_part<PAST>(out + w[u].at, VEC, o);
            }
        };
        int i0 = 0;
        for (; i0 + STEP * AT_ONCE <= n; i0 += STEP * AT_ONCE) take(i0 + threadIdx.x * VEC, true);
        if (i0 < n) take(i0 + threadIdx.x * VEC, false);
    }
}

// How long rows are cut. A workgroup takes a whole row, which saves k_tokens_join and its launch, where that still fills the
// card or the row is short; us for bf16 without and with 20 alternatives:
//   64 threads, many short rows (4 KB; 12 KB from 2,048 rows, 20 KB from 4,096): 8,192 x 1,500 9.6 and 18.5, on 256 threads
//     18.3 and 39.4; 4,096 x 8,000 15.9 and 33.1, 16.7 and 31.9; 2,048 x 12,000 14.9 and 33.6, 12.4 and 22.9
//   256, up to 40 KB: 1 x 5,000 3.0 and 5.8, in segments 4.5 and 10.6; 1,024 x 20,000 10.3 and 17.8, in four 17.7 and 33.2
//   512, up to 64 KB, 128 KB from 96 rows, any from 384: 256 x 60,000 8.9 and 15.9, in four segments 11.8 and 21.5; 512 x
//     131,072 28.3 and 38.7, in three 31.1 and 53.6; but 300 x 131,072 25.9 and 34.8, in four 21.8 and 33.9
//   256 again from 768 rows up to 160 KB: 1,200 x 60,000 31.6 and 47.6, on 512 36.0 and 51.8; 2,000 x 131,072 101 and 151,
//     95 and 131
//   else segments of 256 threads, equally long, at most 64 (the join's lanes): up to two workgroups a CU of a vector a thread
//     at least, up to four of a round at least: 128 x 250,000 18.9 and 30.4 at 1,024 workgroups, 21.8 and 37.7 at 512, 20.1 and
//     34.7 at 1,536; 70 x 131,072 10.4 and 18.5 at 980, 11.3 and 19.7 at 1,050; 16 x 60,000 5.4 and 11.5 at 16 segments, 5.8 and
//     11.7 at 32; 3 x 131,072 4.9 and 10.8 at 42, 5.3 and 11.8 at 21
struct Cut {
    int part, splits, seg;        // threads, segments a row, entries of one
};
inline Cut cut_of(int64_t rows, int vocab, int type) {
    const int64_t size = type == D1_FP32 ? 4 : 2, bytes = vocab * size;
    if (bytes <= (rows >= 4096 ? 20 : rows >= 2048 ? 12 : 4) << 10) return {64, 1, vocab};
    if (bytes <= 40 << 10) return {256, 1, vocab};
    if (bytes <= 64 << 10 || (rows >= 96 && bytes <= 128 << 10) || rows >= 384)
        return {rows >= 768 && bytes <= 160 << 10 ? 256 : 512, 1, vocab};
    const auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
    const int64_t step = 256 * (16 / size), few = least(512 / rows, (vocab + step - 1) / step);
    const int64_t many = least(1024 / rows, vocab / (step * AT_ONCE)), splits = least(few > many ? few : many, 64);
    const int seg = (int)(((vocab + splits - 1) / splits + 7) / 8 * 8);
    return {256, (vocab + seg - 1) / seg, seg};
}
inline unsigned blocks_of(int64_t units) { return (unsigned)(units < (1 << 20) ? units : (1 << 20)); }

// Lanes a row and chunks of four a lane for short rows: several rows a wave and several chunks a lane, since reductions over
// lanes cost as much as the entries (83,378 x 189 bf16: 12.4 us on 16 lanes x 4 chunks, 21.3 on 64 x 1; 62,655 x 89 with 20
// alternatives 34 on 8 x 4, 111 on 64 x 1; 30,000 x 500 fp32 with 5 24.5 on 32 x 4, 41 on 64 x 4; 65,536 x 25 with 3 and a
// mask 6.4 on 8 x 1, 9.7 on 16 x 1).
#define D1O_SMALL_SHAPES(X) X(4, 1) X(8, 1) X(8, 2) X(8, 4) X(16, 4) X(32, 4)

template <class T, bool MASK>
int small_fwd(const Args &a, hipStream_t s) {
#define X(L, C)                                                                                                   \
    if (a.vocab <= L * C * 4) {                                                                                   \
        k_tokens_small<T, L, C, MASK><<<blocks_of((a.rows + 256 / L - 1) / (256 / L)), 256, 0, s>>>(a);           \
        return (int)hipGetLastError();                                                                            \
    }
    D1O_SMALL_SHAPES(X)
#undef X
    return D1_E_ARG;
}
template <class T, bool MASK>
int small_bwd(const BackArgs &a, hipStream_t s) {
#define X(L, C)                                                                                                   \
    if (a.vocab <= L * C * 4) {                                                                                   \
        k_tokens_small_bwd<T, L, C, MASK><<<blocks_of((a.rows + 256 / L - 1) / (256 / L)), 256, 0, s>>>(a);       \
        return (int)hipGetLastError();                                                                            \
    }
    D1O_SMALL_SHAPES(X) X(64, 4)       // no sums over lanes here: wider rows too
#undef X
    return D1_E_ARG;
}

template <class T, bool MASK>
int fwd(const Args &a, const Parts &p, hipStream_t s) {
    if (a.vocab <= SMALL_VOCAB) return small_fwd<T, MASK>(a, s);
    const unsigned grid = blocks_of(a.rows * p.splits);
#define X(P)                                                              \
    if (p.part == P && a.top)                                             \
        k_tokens_part<T, P, MASK, true><<<grid, P, 0, s>>>(a, p);         \
    else if (p.part == P)                                                 \
        k_tokens_part<T, P, MASK, false><<<grid, P, 0, s>>>(a, p);
    X(64) X(256) X(512)
#undef X
    const int e = (int)hipGetLastError();
    if (e || p.splits == 1) return e;
    k_tokens_join<T><<<blocks_of(a.rows), 64, 0, s>>>(a, p);
    return (int)hipGetLastError();
}
template <class T, bool MASK>
int bwd(const BackArgs &a, hipStream_t s) {
    if (a.vocab <= SMALL_BWD_VOCAB) return small_bwd<T, MASK>(a, s);
    // Results that the last cache (256 MB) does not hold go past the caches, a wave a round of one (4,096 x 131,072 bf16 343 us,
    // 348 on 256 threads, 367 there with two rounds; 4,096 x 131,071 377, 412 and 436) or of a row up to two (100,000 x 1,100
    // 83 whole, 108 in rounds). Others stay where the next kernel reads them (16,000 x 4,000 42 us, 51 past the caches; 1,024 x
    // 50,000 fp32 71 and 67).
    // Of those, many rows go whole to 64 threads up to 8 KB (20,000 x 1,100 20.5, on 256 34; 16,000 x 4,001 46.5 and 56) or 256
    // up to 32 KB (8,000 x 9,000 47, in two-round segments 62); longer rows take two rounds a workgroup (1,024 x 50,000 33.8, one
    // round 35.9, four 39.9), where there are few one (300 x 60,001 13.4, two 14.8; 300 x 131,072 27.8 and 26.4).
    const int64_t size = sizeof(T), bytes = a.vocab * size;
    const bool past = a.rows * bytes > 8 * PAST_BYTES, whole = past ? bytes <= 4 << 10 : a.rows >= 1024 && bytes <= 32 << 10;
    const int round = AT_ONCE * (past ? 64 : 256) * (16 / (int)size);
    const int seg = whole ? a.vocab : past || a.rows < 512 ? round : 2 * round;
    const int splits = (a.vocab + seg - 1) / seg;
    const unsigned grid = blocks_of(a.rows * splits);
    if (past)
        k_tokens_bwd<T, 64, MASK, true><<<grid, 64, 0, s>>>(a, splits, seg);
    else if (whole && bytes <= 8 << 10)
        k_tokens_bwd<T, 64, MASK, false><<<grid, 64, 0, s>>>(a, splits, seg);
    else
        k_tokens_bwd<T, 256, MASK, false><<<grid, 256, 0, s>>>(a, splits, seg);
    return (int)hipGetLastError();
}

}  // namespace d1o

using namespace d1o;

#define D1O_TOKEN_TYPES(F, ...)                                                              \
    if (type == D1_FP32) return mask ? F<float, true>(__VA_ARGS__) : F<float, false>(__VA_ARGS__);   \
    if (type == D1_BF16) return mask ? F<__bf16, true>(__VA_ARGS__) : F<__bf16, false>(__VA_ARGS__); \
    return mask ? F<_Float16, true>(__VA_ARGS__) : F<_Float16, false>(__VA_ARGS__);

static bool token_args(int type, int64_t rows, int vocab, int64_t stride, int64_t mask_stride) {
    return is_type(type) && rows >= 0 && vocab >= 1 && vocab <= D1_TOKENS_MAX_VOCAB && stride >= 0 && mask_stride >= 0;
}

extern "C" int64_t d1_tokens_work_bytes(int64_t rows, int vocab, int top) {
    if (!token_args(D1_FP32, rows, vocab, 0, 0) || top < 0 || top > D1_TOKENS_MAX_TOP || top > vocab) return D1_E_ARG;
    if (vocab <= SMALL_VOCAB || rows == 0) return 0;
    const int splits = cut_of(rows, vocab, D1_FP32).splits;      // no type has more
    return splits == 1 ? 0 : rows * splits * (16 + 8 * (int64_t)top);
}

extern "C" int d1_tokens_fwd(const void *logits, int type, int64_t rows, int vocab, int64_t stride, const int64_t *tokens,
                             const uint8_t *mask, int64_t mask_stride, int top, float *logp, float *entropy, float *stats,
                             int64_t *top_ids, float *top_logp, void *work, int64_t work_bytes, void *stream) {
    if (!token_args(type, rows, vocab, stride, mask_stride)) return D1_E_ARG;
    if (top < 0 || top > D1_TOKENS_MAX_TOP || top > vocab) return D1_E_ARG;
    if (rows == 0) return 0;
    if (!logits || !tokens || !logp || !entropy || !stats || (top && (!top_ids || !top_logp))) return D1_E_ARG;
    const int64_t need = d1_tokens_work_bytes(rows, vocab, top);
    if (need && (!work || work_bytes < need || ((uintptr_t)work & 7))) return D1_E_ARG;
    Parts p{};
    if (vocab > SMALL_VOCAB) {
        const Cut c = cut_of(rows, vocab, type);
        p.part = c.part;
        p.splits = c.splits;
        p.seg = c.seg;
        if (p.splits > 1) {
            p.keys = (uint64_t *)work;
            p.sums = (float *)(p.keys + rows * p.splits * top);
        }
    }
    const Args a{logits, rows, stride, vocab, top, tokens, mask, mask_stride, logp, entropy, stats, top_ids, top_logp};
    D1O_TOKEN_TYPES(fwd, a, p, (hipStream_t)stream)
}

extern "C" int d1_tokens_bwd(const void *logits, int type, int64_t rows, int vocab, int64_t stride, const int64_t *tokens,
                             const uint8_t *mask, int64_t mask_stride, const float *stats, const float *entropy,
                             const float *dlogp, const float *dentropy, void *dlogits, void *stream) {
    if (!token_args(type, rows, vocab, stride, mask_stride)) return D1_E_ARG;
    if (rows == 0) return 0;
    if (!logits || !tokens || !stats || !dlogits || dlogits == logits || (dentropy && !entropy)) return D1_E_ARG;
    const BackArgs a{logits, rows, stride, vocab, tokens, mask, mask_stride, stats, entropy, dlogp, dentropy, dlogits};
    D1O_TOKEN_TYPES(bwd, a, (hipStream_t)stream)
}
