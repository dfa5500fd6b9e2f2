// What the block seam (block_seam.hip) and its gradients (block_seam_grad.hip)
// share: how rows and columns are laid over lanes, loads, and row sums.
//
// A thread owns C times 8 columns and keeps their parameters, and in the
// gradients their column sums, in registers while it walks down the rows of a
// sequence.  A row is taken by L lanes of a wave (8, 16, 32 or 64: up to 512
// columns; its sums are butterflies in registers), or by the whole block (L = 0:
// the waves' sums meet in LDS, one barrier for the rows of a step).
#pragma once

#include "kernels.hpp"
#include "seam.hpp"

namespace nomas {

constexpr int kSeamCols = 8;          // columns of one chunk (D % 8 == 0)
constexpr int kSeamNarrow = 256;      // threads of a block whose rows take a wave's lanes
constexpr int kSeamWide = 512;        // and at most, where a row takes the block
constexpr int kSeamStep = 2;          // rows of a group that the plan counts to a step

// The rows of a call over the grid.
//  whole == 0: `parts` blocks share each sequence, `chunk` rows a block
//  whole != 0: each group of lanes takes whole sequences in turn
struct SeamPlan {
    int L, C, threads, groups;  // lanes per row (0: the block), chunks per thread
    int whole;
    int64_t blocks, parts, chunk;
};

// `target`: blocks that fill the chip.  Sequences are shared by blocks unless
// they are shorter than two steps or there are enough of them to fill the chip.
inline SeamPlan seam_plan(int64_t rows, int64_t D, int64_t seq, int64_t target) {
    SeamPlan p{};
    const int64_t chunks = D / kSeamCols;
    p.L = chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : chunks <= 64 ? 64 : 0;
    p.C = p.L || chunks <= kSeamWide ? 1 : chunks <= 2 * kSeamWide ? 2 : 4;
    p.threads = p.L ? kSeamNarrow : (int)round_up((chunks + p.C - 1) / p.C, kWave);
    p.groups = p.L ? kSeamNarrow / p.L : 1;
    const int64_t n = rows / seq, step = (int64_t)p.groups * kSeamStep;
    p.whole = seq < 2 * step || n >= target * p.groups;
    if (p.whole) {
        p.parts = 1;
        p.chunk = seq;
        p.blocks = (n + p.groups - 1) / p.groups;
        if (p.blocks > target) p.blocks = target;
        return p;
    }
    p.parts = (target + n - 1) / n;
    if (p.parts > (seq + step - 1) / step) p.parts = (seq + step - 1) / step;
    p.chunk = round_up((seq + p.parts - 1) / p.parts, step);
    p.parts = (seq + p.chunk - 1) / p.chunk;
    p.blocks = n * p.parts;
    return p;
}

// Eight elements of a row as loaded.
template <typename T> struct Raw8 {
    uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> fetch8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float* o) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) unpack16<T>(r.v[i], o + i * (16 / sizeof(T)));
}
template <typename T>
__device__ __forceinline__ void put8(T* p, const float* v) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) store16(p + i * (16 / sizeof(T)), v + i * (16 / sizeof(T)));
}
// eight f32 parameters, or `other` where there are none
__device__ __forceinline__ void params8(const float* p, int64_t at, float other, float* o) {
    if (p) {
        load_f32s<8>(p + at, o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = other;
    }
}

template <int kCtrl>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
}

// The sum over each L neighbouring lanes, in all of them.
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
    v = dpp_add<0xb1>(v);                    // quad_perm: lane ^ 1
    v = dpp_add<0x4e>(v);                    // quad_perm: lane ^ 2
    v = dpp_add<0x141>(v);                   // row_half_mirror: the other four of eight
    if constexpr (L >= 16) v = dpp_add<0x140>(v);  // row_mirror: the other eight of sixteen
    if constexpr (L >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if constexpr (L >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}

// The sums of N values over a row's lanes, in all of them.  L = 0: over the
// block; `part` [2][8 waves][N] takes turns by `turn`, so that one barrier a call
// is enough.
template <int L, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* part, int turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane_sum<L ? L : 64>(v[i]);
    if constexpr (L == 0) {
        float* p = part + (turn & 1) * (kSeamWide / kWave) * N;
        const int wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) p[wave * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = p[i];
        for (int w = 1; w < nw; ++w)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += p[w * N + i];
    }
}

// Calls f with a plan's L and C as constants.
template <typename F>
hipError_t with_seam_shape(const SeamPlan& p, F f) {
    using std::integral_constant;
    switch (p.L) {
        case 8: return f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
        case 16: return f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
        case 32: return f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
        case 64: return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    }
    switch (p.C) {
        case 1: return f(integral_constant<int, 0>{}, integral_constant<int, 1>{});
        case 2: return f(integral_constant<int, 0>{}, integral_constant<int, 2>{});
    }
    return f(integral_constant<int, 0>{}, integral_constant<int, 4>{});
}

}  // namespace nomas
