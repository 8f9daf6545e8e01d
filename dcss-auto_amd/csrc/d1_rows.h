// d1ops: what the row operators (d1_tokens.hip, d1_norm.hip) and the AdamW step (d1_optim.hip) share:
// packs of adjacent elements and reductions over 1 to 64 lanes, gfx950.
#ifndef D1_ROWS_H
#define D1_ROWS_H
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/d1ops.h"
#include "d1_frag.h"

namespace d1o {

// N adjacent elements, loaded and stored whole from any element-aligned address (global memory
// takes unaligned 16-byte accesses, so odd row lengths need no path of their own)
template <class T, int N>
struct Pack {
    T v[N];
};
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load(const T *p) {
    Pack<T, N> a;
    __builtin_memcpy(&a, p, sizeof a);
    return a;
}
template <class T, int N>
__device__ __forceinline__ void store(T *p, const Pack<T, N> &a) {
    __builtin_memcpy(p, &a, sizeof a);
}
// the first n (0 to N) of them; the others read as `fill` and are not written
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_part(const T *p, int n, T fill) {
    if (n >= N) return load<T, N>(p);
    Pack<T, N> a;
#pragma unroll
    for (int i = 0; i < N; i++) a.v[i] = i < n ? p[i] : fill;
    return a;
}
template <class T, int N>
__device__ __forceinline__ void store_part(T *p, int n, const Pack<T, N> &a) {
    if (n >= N) return store<T, N>(p, a);
#pragma unroll
    for (int i = 0; i < N; i++)
        if (i < n) p[i] = a.v[i];
}

// A lane's pack of elements i to i + N - 1 of n, moved back where it would pass the end: one whole load without a
// branch, of which the first `skip` elements are the lanes' before it (all N of them where i >= n). Both lanes store
// the same values there. There have to be N elements before the end.
struct Place {
    int at, skip;
};
template <int N>
__device__ __forceinline__ Place place_of(int i, int n) {
    const int at = i < n - N ? i : n - N;
    return {at, i - at};
}

// the same past the caches, for outputs that are larger than the L2s of all chiplets (8 x 4 MB) and so
// would only push out what is read
constexpr int64_t PAST_BYTES = 32 << 20;
template <class T, int N>
__device__ __forceinline__ void store_past(T *p, const Pack<T, N> &a) {
    constexpr int WORDS = (int)sizeof(a) / 4;
    static_assert(WORDS == 1 || WORDS == 2 || WORDS == 4, "one store instruction");
    if constexpr (WORDS == 1) {
        typedef uint32_t anywhere __attribute__((aligned(1)));
        __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, a), (anywhere *)p);
    } else {
        typedef uint32_t words __attribute__((ext_vector_type(WORDS)));
        typedef words anywhere __attribute__((aligned(1)));
        __builtin_nontemporal_store(__builtin_bit_cast(words, a), (anywhere *)p);
    }
}
template <bool PAST, class T, int N>
__device__ __forceinline__ void put_part(T *p, int n, const Pack<T, N> &a) {
    if (PAST && n >= N)
        store_past<T, N>(p, a);
    else
        store_part<T, N>(p, n, a);
}

// op over aligned groups of LANES lanes (1, 2, 4 ... 64); every lane gets the same result: partners
// at distance 1, 2, 4, 8 through DPP, 16 and 32 through the lane-swap moves. After the steps before,
// the lanes of a quad (of a half row) hold equal values, so a mirror reads the other quad's (half's).
constexpr int DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
template <int LANES, class Op>
__device__ __forceinline__ uint32_t lanes_u(uint32_t x, Op op) {
    if (LANES > 1) x = op(x, dpp_u<d1f::DPP_XOR1>(x));
    if (LANES > 2) x = op(x, dpp_u<d1f::DPP_XOR2>(x));
    if (LANES > 4) x = op(x, dpp_u<DPP_HALF_MIRROR>(x));
    if (LANES > 8) x = op(x, dpp_u<DPP_MIRROR>(x));
    if (LANES > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        const uint32_t a = r[0], b = r[1];
        x = op(a, b);
    }
    if (LANES > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        const uint32_t a = r[0], b = r[1];
        x = op(a, b);
    }
    return x;
}
template <int LANES, class Op>
__device__ __forceinline__ float lanes_f(float x, Op op) {
    return __uint_as_float(lanes_u<LANES>(__float_as_uint(x), [&](uint32_t a, uint32_t b) {
        return __float_as_uint(op(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
    return lanes_f<LANES>(x, [](float a, float b) { return a + b; });
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float x) {
    return lanes_f<LANES>(x, [](float a, float b) { return fmaxf(a, b); });
}

inline bool is_type(int t) { return t == D1_FP32 || t == D1_BF16 || t == D1_FP16; }

}  // namespace d1o
#endif
