// What the block seam (block_seam.hip) and its gradients (block_seam_grad.hip)
// share: how rows and columns are laid over lanes, loads, and row sums.
//
// A thread owns C times 8 columns and keeps their parameters, and in the
// gradients their column sums, in registers while it walks down the rows of a
// sequence.  A row is taken by L lanes of a wave (8, 16, 32 or 64: up to 512
// columns; its sums are made in registers), or by several waves (L = 0: their sums
// meet in LDS, one barrier for the rows of a step).
#pragma once

#include "kernels.hpp"
#include "seam.hpp"

namespace nomas {

constexpr int kSeamCols = 8;          // columns of one chunk (D % 8 == 0)
constexpr int kSeamThreads = 512;     // of a block, at most
constexpr int kSeamWaves = kSeamThreads / kWave;
constexpr int kSeamStep = 2;          // rows of a group that the plan counts to a step

// The rows of a call over the grid.  A block has `groups` of `row_threads`
// threads, each of which takes a row at a time.
//  whole == 0: `parts` blocks share each sequence, `chunk` rows a block
//  whole != 0: each group takes whole sequences in turn
struct SeamPlan {
    int L, C, row_threads, groups;  // L: lanes per row, 0 where a row takes several waves
    int whole;
    int64_t blocks, parts, chunk;
};

// `target`: blocks that fill the chip; `most`: threads of a block (a row may need
// more).  Sequences are shared by blocks unless they are shorter than two rows of
// each group or there are enough of them to fill the chip.  A few short sequences of narrow rows are then
// walked row by row by a group each, with most of the chip idle: 191 rows of 64 take 160 us in the gradients,
// 47 of 256 45, 8 x 11 of 1,024 19; in the forward pass 127 rows of 64 take 54 us.
inline SeamPlan seam_plan(int64_t rows, int64_t D, int64_t seq, int64_t target, int most) {
    SeamPlan p{};
    const int64_t chunks = D / kSeamCols;
    p.L = chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : chunks <= 64 ? 64 : 0;
    p.C = p.L || chunks <= kSeamThreads ? 1 : chunks <= 2 * kSeamThreads ? 2 : 4;
    p.row_threads = p.L ? p.L : (int)round_up((chunks + p.C - 1) / p.C, kWave);
    p.groups = p.row_threads < most ? most / p.row_threads : 1;
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
// Likewise `col` elements from a row: a base that is the same for a wave stays in
// scalar registers, the lane's offset is 32 bits.
template <typename T>
__device__ __forceinline__ Raw8<T> fetch8(const T* row, uint32_t col) {
    return fetch8(reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + col * (uint32_t)sizeof(T)));
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
// Hides from the compiler that it has widened these elements before, so that it
// widens them again (an instruction each) instead of keeping the f32 values.
template <typename T>
__device__ __forceinline__ void renew(Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        asm("" : "+v"(r.v[i].x), "+v"(r.v[i].y), "+v"(r.v[i].z), "+v"(r.v[i].w));
}
template <typename T>
__device__ __forceinline__ void put8(T* row, uint32_t col, const float* v) {
    put8(reinterpret_cast<T*>(reinterpret_cast<char*>(row) + col * (uint32_t)sizeof(T)), v);
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

// The sum over each L <= 32 neighbouring lanes, in all of them.
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
    return v;
}

// The wave's sums of a, b, c, d: in its lanes 0-15 a's, 16-31 c's, 32-47 b's, 48-63
// d's.  Halves and rows of lanes are exchanged between the values instead of
// being added for each: ten instructions for four sums.
__device__ __forceinline__ float four_sums(float a, float b, float c, float d) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(c), __float_as_uint(d), false, false);
    const float ab = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    const float cd = __uint_as_float(q[0]) + __uint_as_float(q[1]);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(ab), __float_as_uint(cd), false, false);
    float v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    v = dpp_add<0xb1>(v);
    v = dpp_add<0x4e>(v);
    v = dpp_add<0x141>(v);
    return dpp_add<0x140>(v);
}

// LDS floats of row_sums for N values a row: two turns of all waves' sums, four
// values in 16 bytes.
template <int L, int N>
constexpr int sums_floats() { return L ? 1 : 2 * kSeamWaves * ((N + 3) / 4 * 4); }

// The sums of N values over a row's lanes, in all of them.  L = 0: over the
// row's waves; `part` takes turns by `turn`, so that one barrier a call is enough.
template <int L, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* part, int turn, int row_waves) {
    if constexpr (L > 0 && L < 64) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lane_sum<L>(v[i]);
        return;
    } else {
        constexpr int Q = (N + 3) / 4;
        float s[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i)
            s[i] = four_sums(v[4 * i], 4 * i + 1 < N ? v[min(4 * i + 1, N - 1)] : 0.0f,
                             4 * i + 2 < N ? v[min(4 * i + 2, N - 1)] : 0.0f,
                             4 * i + 3 < N ? v[min(4 * i + 3, N - 1)] : 0.0f);
        auto at = [](int i) { return (i & 1) * 32 + (i & 2) * 8; };  // lane of the i-th of four
        if constexpr (L == 64) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                v[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s[i / 4]), at(i & 3)));
            return;
        }
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        float* p = part + (turn & 1) * kSeamWaves * 4 * Q;
        if ((lane & 15) == 0) {
            const int slot = (lane >> 5) + ((lane >> 4) & 1) * 2;
#pragma unroll
            for (int i = 0; i < Q; ++i) p[(wave * Q + i) * 4 + slot] = s[i];
        }
        __syncthreads();
        const float4* first = reinterpret_cast<const float4*>(p) + wave / row_waves * row_waves * Q;
        float4 t[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) t[i] = first[i];
        for (int w = 1; w < row_waves; ++w)
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const float4 o = first[w * Q + i];
                t[i].x += o.x;
                t[i].y += o.y;
                t[i].z += o.z;
                t[i].w += o.w;
            }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i % 4 == 0 ? t[i / 4].x : i % 4 == 1 ? t[i / 4].y : i % 4 == 2 ? t[i / 4].z : t[i / 4].w;
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
