// The MoE layer on up to 64 rows: gate/up with SwiGLU, then down with the weighted sum, each one
// kernel over all chosen experts.
//
//   h[e, r] = silu(x_r Wg_e^T + bg_e) (x_r Wu_e^T + bu_e)         for the rows r that chose e
//   y_r     = sum over the chosen e, ascending, of w[r, e] (h[e, r] Wd_e^T + bd_e)
//
// What bounds such a call is the chosen experts' weights on their way from HBM, and for the
// smallest ones the launches.  So there is no dispatch: as a block starts, it makes the lists of
// the rows that chose each expert from the routing (a 64-bit mask per expert), and reads
// rows where they are; and no combine: a block of the second kernel has a tile of 16
// columns for all rows and experts, or shares it with a few others.  Weights are read in the layouts that
// the layer keeps (K-blocked, kernels.hpp), a 16 x 16-byte fragment of an MFMA per instruction, straight
// into registers, or as 8-bit values in fragment order, widened there.
//
// h is rounded to the layer's type, in which the second kernel's MFMAs take it and in which the layer's
// forward of many rows keeps it (an output's error is then 1.4 times that of its own rounding);
// y's sums stay f32 over all experts and are rounded once.
#include "fp8.hpp"
#include "mfma.hpp"

#include <algorithm>

namespace nomas {

namespace {

constexpr int kFewThreads = 512;
constexpr int kFewWaves = kFewThreads / kWave;

// Fragments of a step of KS columns: two of 16 weight rows x 64 bytes, XL of 16 token rows x 16 bytes
// a lane.  xk: the lane's column of the q-th token fragment in a step.
template <typename T, bool W8> struct Step {
    static constexpr int KS = W8 ? 128 : 128 / (int)sizeof(T), XL = W8 ? 4 : 2, CH = 16 / (int)sizeof(T);
    static __device__ __forceinline__ int xk(int q, int lq) {
        return W8 ? q / 2 * 64 + lq * 16 + q % 2 * 8 : q * (KS / 2) + lq * CH;
    }
};

// 8-bit weights as 16-bit values, and what those are short of the weights' scale `s`: v * rest = w * s.  A block's
// sum of bf16 rows by weights of up to 448 leaves f32 from 2^112 on, where its product with a scale below 1 does
// not: such weights are taken times 2^-16 (and stay normal bf16 numbers), so that no sum can.  A scale from 1 on makes
// the sum larger still.  f16 rows end at 2^16.
template <typename T> struct Widen8;
template <> struct Widen8<__bf16> {
    typedef __bf16 V2 __attribute__((ext_vector_type(2)));
    float down, rest;
    __device__ __forceinline__ explicit Widen8(float s) {
        const bool less = __builtin_fabsf(s) < 1.0f;
        down = less ? 0x1p-16f : 1.0f;
        rest = less ? s * 0x1p16f : s;
    }
    __device__ __forceinline__ V2 run(uint32_t w, bool hi) const {
        return hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, down, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, down, false);
    }
};
template <> struct Widen8<_Float16> {
    typedef _Float16 V2 __attribute__((ext_vector_type(2)));
    float rest;
    __device__ __forceinline__ explicit Widen8(float s) : rest(s) {}
    __device__ __forceinline__ V2 run(uint32_t w, bool hi) const {
        return hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false);
    }
};

// The rows' fragments of a step, 16 J rows.
template <typename T, bool W8, int J> struct Rows {
    u32x4_t x[J][Step<T, W8>::XL];
};

// acc += the step's products.  `s`: the scale of 8-bit weights, else what f32 weights are taken down by.
template <typename T, bool W8, int J>
__device__ __forceinline__ void multiply(f32x4_t* acc, const u32x4_t (&w)[2], const u32x4_t (*x)[Step<T, W8>::XL], float s) {
    if constexpr (W8) {
        typedef typename Mfma<T>::V V;
        const Widen8<T> to16(s);
        V a[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const auto v = to16.run(w[q / 2][q % 2 * 2 + i], h);
                    a[q][i * 4 + h * 2] = v[0];
                    a[q][i * 4 + h * 2 + 1] = v[1];
                }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            f32x4_t t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < 4; ++q) t = Mfma<T>::run(a[q], __builtin_bit_cast(V, x[j][q]), t);
            // The result is there 8 wait states after the last MFMA.  The compiler moved its use behind a
            // branch that skipped the next rows' products and counted the waits along the longer
            // way only: every fourth column was wrong.  So the wait stands here.
            asm volatile("s_nop 8" : "+v"(t));
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j][r] = __builtin_fmaf(t[r], to16.rest, acc[j][r]);
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = __uint_as_float(w[q][k]) * s;
#pragma unroll
                for (int j = 0; j < J; ++j) acc[j] = mfma_f32(v, __uint_as_float(x[j][q][k]), acc[j]);
            }
    } else {
        typedef typename Mfma<T>::V V;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int j = 0; j < J; ++j)
                acc[j] = Mfma<T>::run(__builtin_bit_cast(V, w[q]), __builtin_bit_cast(V, x[j][q]), acc[j]);
    }
}

// f(J) with 16 J >= n rows, J of 1, 2, 4 up to NT: code with the loads ahead that so few rows leave registers for.
template <int NT, typename F>
__device__ __forceinline__ void for_rows(int n, F f) {
    using std::integral_constant;
    if (NT == 1 || n <= 16) f(integral_constant<int, 1>{});
    else if (NT == 2 || n <= 32) f(integral_constant<int, NT < 2 ? NT : 2>{});
    else f(integral_constant<int, NT>{});
}

__device__ __forceinline__ u32x4_t load16u(const void* p) { return *reinterpret_cast<const u32x4_t*>(p); }

// Who has chosen, or will (FewArgs::choice): a kernel before or the caller, or the first kernel, from
// logits or from the rows themselves.
enum { kChoiceMade = 0, kChoiceOfLogits = 1, kChoiceOfRows = 2 };

// ---- the router's choice ---------------------------------------------------------
// Softmax over the logits, top-k with ties to the lowest index, weights p / (sum of the chosen p + 1e-9)
// in ascending order of experts: the layer's router (router.hip) for few rows.  16-bit products are exact
// in f32, each MFMA's 32 of them summed there and those sums in f64; f32 inputs take f64 MFMAs.

typedef double d4_t __attribute__((ext_vector_type(4)));

// The logits of 16 rows and 16 experts, D shared by the block's waves; thread t < 256 returns that of
// row t / 16 and expert t % 16.  s_part: 256 per wave.
template <typename T>
__device__ __forceinline__ double logit_tile(const FewArgs& a, int rg, int eg, double* s_part) {
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int CH = 16 / (int)sizeof(T), KS = 4 * CH;  // columns a lane, and of a step
    const int steps = (a.D + KS - 1) / KS, s0 = steps * wave / kFewWaves, s1 = steps * (wave + 1) / kFewWaves;
    const T* x = static_cast<const T*>(a.x) + (int64_t)min(rg * 16 + l16, a.rows - 1) * a.D + lq * CH;
    const T* w = static_cast<const T*>(a.wr) + (int64_t)min(eg * 16 + l16, a.E - 1) * a.D + lq * CH;
    d4_t acc = {0.0, 0.0, 0.0, 0.0};
    constexpr int U = 8;
    for (int st = s0; st < s1; st += U) {
        u32x4_t xv[U], wv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (st + u) * KS;
            xv[u] = wv[u] = u32x4_t{0, 0, 0, 0};
            if (st + u < s1 && k + lq * CH < a.D) {
                xv[u] = load16u(x + k);
                wv[u] = load16u(w + k);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {  // (past the end: zeros)
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)__uint_as_float(xv[u][i]),
                                                               (double)__uint_as_float(wv[u][i]), acc, 0, 0, 0);
            } else {
                typedef typename Mfma<T>::V V;
                const f32x4_t z = {0.0f, 0.0f, 0.0f, 0.0f};
                const f32x4_t t = Mfma<T>::run(__builtin_bit_cast(V, xv[u]), __builtin_bit_cast(V, wv[u]), z);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] += (double)t[r];
            }
        }
    }
    // lane: expert l16 of rows 4 lq + r (f64 MFMAs: lq + 4 r)
#pragma unroll
    for (int r = 0; r < 4; ++r) s_part[wave * 256 + (sizeof(T) == 4 ? lq + 4 * r : 4 * lq + r) * 16 + l16] = acc[r];
    __syncthreads();
    double v = 0.0;
    if (tid < 256) {
        v = s_part[tid];
#pragma unroll
        for (int i = 1; i < kFewWaves; ++i) v += s_part[i * 256 + tid];
    }
    return v;
}

// f64 as an integer of the same order; NaN above all, so that the choice is always k experts.
__device__ __forceinline__ int64_t order_key(double v) {
    if (v != v) return INT64_MAX;
    const int64_t b = __double_as_longlong(v + 0.0);  // (-0 is 0)
    return b ^ ((b >> 63) & 0x7fffffffffffffffll);
}
template <int kCtrl>
__device__ __forceinline__ float dpp_addf(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
}
// Over a wave, in all lanes.
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_addf<0xb1>(v);
    v = dpp_addf<0x4e>(v);
    v = dpp_addf<0x141>(v);
    v = dpp_addf<0x140>(v);
    auto lane = [&](int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)); };
    return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

__device__ __forceinline__ uint32_t wave_maxu(uint32_t v) {
    const uint32_t m = max16(v);
    auto lane = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)m, i); };
    return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}
// f32 bits as an unsigned integer of the same order, NaN above all.
__device__ __forceinline__ uint32_t order_key32(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}

// Which of the lane's experts (bit j: lane + 64 j) are among the k of the largest logits, ties to the lowest
// index.  By the logits as f32, whose order is that of f64 but for equal ones, and by f64 where more than
// one choice is possible so.  Up to 64 experts: each lane counts those above its own; more: the k-th
// value by bisection over its bits.  s_key: 64 words of the wave's.  (64-bit compares of all
// with all took 4.5 us for one row of 64 experts.)
template <int PL>
__device__ __forceinline__ uint32_t choose_largest(const double* l, const double (&v)[PL], int E, int k, uint32_t* s_key) {
    const int lane = threadIdx.x & 63;
    uint32_t key[PL], mine = 0;
    int count = 0;
#pragma unroll
    for (int j = 0; j < PL; ++j) key[j] = lane + j * 64 < E ? order_key32((float)v[j]) : 0u;  // (0: below all)
    if constexpr (PL == 1) {
        s_key[lane] = key[0];  // (one wave: its LDS accesses are in order)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        int above = 0;
        for (int e = 0; e < E; e += 16) {
            u32x4_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = *reinterpret_cast<const u32x4_t*>(s_key + e + i * 4);
#pragma unroll
            for (int i = 0; i < 16; ++i) above += o[i / 4][i % 4] > key[0] ? 1 : 0;
        }
        mine = lane < E && above < k ? 1u : 0u;
        count = __popcll(__ballot(mine));
    } else {
        uint32_t kth = 0;  // the largest value that at least k are not below
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < PL; ++j) n += __popcll(__ballot(key[j] >= (kth | bit)));
            if (n >= k) kth |= bit;
        }
#pragma unroll
        for (int j = 0; j < PL; ++j) {
            const bool in = key[j] >= kth && lane + j * 64 < E;
            mine |= in ? 1u << j : 0u;
            count += __popcll(__ballot(in));
        }
    }
    if (count == k) return mine;
    mine = 0;
    int64_t own[PL];
    int before[PL];
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        own[j] = order_key(v[j]);
        before[j] = 0;
    }
#pragma unroll 1
    for (int e = 0; e < E; ++e) {
        const int64_t o = order_key(l[e]);
#pragma unroll
        for (int j = 0; j < PL; ++j) before[j] += o > own[j] || (o == own[j] && e < lane + j * 64);
    }
#pragma unroll
    for (int j = 0; j < PL; ++j) mine |= lane + j * 64 < E && before[j] < k ? 1u << j : 0u;
    return mine;
}

// One wave chooses for one row: its logits `l` (LDS, E of them), PL a lane.
template <int PL, typename F>
__device__ __forceinline__ void choose(const FewArgs& a, const double* l, int row, bool store, uint32_t* s_key, F chosen) {
    const int lane = threadIdx.x & 63, E = a.E, k = a.top_k;
    double v[PL];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        const int e = lane + j * 64;
        v[j] = e < E ? l[e] : -INFINITY;
        m = fmaxf(m, (float)v[j]);
    }
    const uint32_t mine = choose_largest<PL>(l, v, E, k, s_key);
    int at = 0, t[PL];
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        const uint64_t c = __ballot(mine >> j & 1);
        t[j] = at + __popcll(c & ((1ull << lane) - 1));  // (places in ascending order of experts)
        at += __popcll(c);
        if (mine >> j & 1) chosen(lane + j * 64);
    }
    if (!store) return;
    // Any number within 1 of the largest does: as f32 up to 2^24, from there on (and past f32) the f64 one,
    // which takes six more shuffles of two words.
    const uint32_t b = wave_maxu(order_key32(m));
    m = __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
    double top = (double)m;
    if (!(__builtin_fabsf(m) < 0x1p24f)) {
        top = v[0];
#pragma unroll
        for (int j = 1; j < PL; ++j) top = fmax(top, v[j]);
#pragma unroll 1
        for (int o = 32; o >= 1; o >>= 1) top = fmax(top, __shfl_xor(top, o));
    }
    float p[PL], sum = 0.0f, sel = 0.0f;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        p[j] = lane + j * 64 < E ? expf((float)(v[j] - top)) : 0.0f;
        sum += p[j];
        sel += mine >> j & 1 ? p[j] : 0.0f;
    }
    sum = wave_sum(sum);
    sel = wave_sum(sel);
    // p / sum / (sel / sum + 1e-9)
    const float norm = 1.0f / (sel + 1e-9f * sum);
    // the last one chosen and the first one not, for the gap between them
    double kth = INFINITY, next = -INFINITY;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        if (mine >> j & 1) {
            a.out_idx[row * a.out_slots + t[j]] = lane + j * 64;
            a.out_w[row * a.out_slots + t[j]] = p[j] * norm;
            kth = fmin(kth, v[j]);
        } else {
            next = fmax(next, v[j]);  // (past E: -infinity)
        }
    }
#pragma unroll 1
    for (int o = 32; o >= 1; o >>= 1) {
        kth = fmin(kth, __shfl_xor(kth, o));
        next = fmax(next, __shfl_xor(next, o));
    }
    if (lane == 0) {
        a.out_gap[row] = k == E ? INFINITY : (float)(kth - next);
        if (a.out_slots > k) {
            a.out_idx[row * a.out_slots + k] = E;
            a.out_w[row * a.out_slots + k] = a.dense_coef;
        }
    }
}
template <typename F>
__device__ __forceinline__ void choose_any(const FewArgs& a, const double* l, int row, bool store, uint32_t* s_key, F chosen) {
    if (a.E <= 64) choose<1>(a, l, row, store, s_key, chosen);
    else choose<kMaxExperts / 64>(a, l, row, store, s_key, chosen);
}

// A kernel of its own: a block for 16 rows and 16 experts; with more than 16 rows in all the last block of each 16
// chooses for them.  Latencies bound it: the router's weights once from HBM, a sum over the waves, the logits' way
// past the caches.  4.6 us for one row of 2,048 and 64 experts, 6.8 for 48 rows of 1,024 and 16.
template <typename T>
__global__ __launch_bounds__(kFewThreads) void few_route_kernel(FewArgs a) {
    extern __shared__ __align__(16) uint8_t s_dyn[];  // 16 rows' logits
    __shared__ double s_part[kFewWaves * 256];
    __shared__ int s_count[kMaxExperts + 1], s_last;
    __shared__ __align__(16) uint32_t s_key[kFewWaves * 64];
    double* s_logit = reinterpret_cast<double*>(s_dyn);
    const int tid = threadIdx.x, wave = tid >> 6, eg = blockIdx.x, rg = blockIdx.y, groups = gridDim.x;
    const double v = logit_tile<T>(a, rg, eg, s_part);
    const int r = tid / 16, e = eg * 16 + tid % 16;
    if (a.choice == kChoiceOfLogits) {  // the first kernel chooses
        if (tid < 256 && e < a.E) a.logits[(rg * 16 + r) * kMaxExperts + e] = v;
        return;
    }
    if (groups > 1) {
        // as in few_down_kernel: past the L2 caches, written before the block is counted
        constexpr int kSc1 = 16;
        const auto rs = __builtin_amdgcn_make_buffer_rsrc(a.logits, 0, kFewRows * kMaxExperts * 8, 0x00020000);
        typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
        if (tid < 256 && e < a.E)
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, v), rs, ((rg * 16 + r) * kMaxExperts + e) * 8, 0,
                                                  kSc1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        int32_t* count = a.arrived + a.tile_cap + rg;
        if (tid == 0)
            s_last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
        __syncthreads();
        if (!s_last) return;
        for (int i = tid; i < 16 * a.E; i += kFewThreads) {
            const int row = i / a.E, ex = i - row * a.E;
            s_logit[i] = __builtin_bit_cast(
                double, __builtin_amdgcn_raw_buffer_load_b64(rs, ((rg * 16 + row) * kMaxExperts + ex) * 8, 0, kSc1));
        }
    } else if (tid < 256 && e < a.E) {
        s_logit[r * a.E + e] = v;
    }
    for (int i = tid; i < a.Ecols; i += kFewThreads) s_count[i] = i < a.E ? 0 : min(16, a.rows - rg * 16);
    __syncthreads();
    for (int i = wave; i < min(16, a.rows - rg * 16); i += kFewWaves)
        choose_any(a, s_logit + i * a.E, rg * 16 + i, true, s_key + wave * 64, [&](int ex) { atomicAdd(&s_count[ex], 1); });
    __syncthreads();
    for (int i = tid; i < a.Ecols; i += kFewThreads) a.out_count[rg * a.Ecols + i] = s_count[i];
}

// What a block knows of the routing.
struct Lists {
    uint64_t* mask;  // [Ecols] rows that chose the expert
    int* live;       // [Ecols] the chosen experts, ascending
    int* off;        // [Ecols] the expert's first place in `row`
    int* info;       // [16] scratch; [0]: chosen experts
    uint8_t* row;    // [places] the experts' rows, one after another
    float* gate;     // ... and their weights (second kernel)
    static __host__ __device__ size_t bytes(int ecols, int places, bool gates) {
        return (size_t)ecols * 16 + 64 + (size_t)(places + 15) / 16 * 16 + (gates ? (size_t)places * 4 : 0);
    }
    // (a multiple of 8 bytes without gates)
    __device__ Lists(uint8_t* p, int ecols, int places) {
        mask = reinterpret_cast<uint64_t*>(p);
        live = reinterpret_cast<int*>(p + (size_t)ecols * 8);
        off = live + ecols;
        info = off + ecols;
        row = reinterpret_cast<uint8_t*>(info + 16);
        gate = reinterpret_cast<float*>(row + (places + 15) / 16 * 16);
    }
};

// The slots of a call in LDS (experts, weights); calls of more of them are read again where needed.
constexpr int kStaged = 2048;

// Experts named twice by a row have the sum of their weights, in the slots' order.
// `logits`: where the routing is still to be chosen (by the first kernel; its block 0 keeps it for the second).
template <bool kGates>
__device__ __forceinline__ void make_lists(const FewArgs& a, const Lists& l, const double* logits = nullptr) {
    __shared__ int16_t s_e[kGates ? kStaged : 1];
    __shared__ float s_w[kGates ? kStaged : 1];
    __shared__ __align__(16) uint32_t s_key[kGates ? 4 : kFewWaves * 64];
    const int tid = threadIdx.x, n = logits ? 0 : a.rows * a.k, lane = tid & 63, wave = tid >> 6;
    const bool staged = n <= kStaged;
    // (on their way while the masks are cleared)
    const int first_e = tid < n ? a.idx[tid] : -1;
    const float first_w = kGates && tid < n ? a.w[tid] : 0.0f;
    for (int e = tid; e < a.Ecols; e += kFewThreads)
        l.mask[e] = e < a.E ? 0 : ~0ull >> (64 - a.rows);  // (the shared branch: all rows)
    __syncthreads();
    for (int i = tid; i < n; i += kFewThreads) {
        const int in = i == tid ? first_e : a.idx[i], e = in >= 0 && in < a.E ? in : -1;
        if (e >= 0) atomicOr(reinterpret_cast<unsigned long long*>(&l.mask[e]), 1ull << (i / a.k));
        if constexpr (kGates)
            if (staged) {
                s_e[i] = (int16_t)e;
                s_w[i] = i == tid ? first_w : a.w[i];
            }
    }
    if constexpr (!kGates) {
        if (logits)
            for (int r = wave; r < a.rows; r += kFewWaves)
                choose_any(a, logits + r * a.E, r, blockIdx.x == 0, s_key + wave * 64, [&](int e) {
                    atomicOr(reinterpret_cast<unsigned long long*>(&l.mask[e]), 1ull << r);
                });
    }
    __syncthreads();
    // places: the chosen experts before, and their rows (512 threads hold all experts)
    static_assert(kMaxExperts + 1 <= kFewThreads, "an expert a thread");
    const uint64_t mine = tid < a.Ecols ? l.mask[tid] : 0;
    const int c = __popcll(mine);
    const uint64_t some = __ballot(c > 0);
    int sum = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 63) l.info[wave] = __popcll(some) << 16 | sum;
    __syncthreads();
    int before = 0, first = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
        const int v = l.info[w];
        all += v >> 16;
        if (w < wave) {
            before += v >> 16;
            first += v & 0xffff;
        }
    }
    if (c > 0) {
        l.live[before + __popcll(some & ((1ull << lane) - 1))] = tid;
        int p = first + sum - c;
        l.off[tid] = p;
        for (uint64_t m = mine; m; m &= m - 1, ++p) {
            l.row[p] = (uint8_t)__builtin_ctzll(m);
            if constexpr (kGates) l.gate[p] = a.dense_coef;  // (of the shared branch; the others' below)
        }
    }
    __syncthreads();
    if (tid == 0) l.info[0] = all;
    if constexpr (kGates) {
        auto expert = [&](int i) {
            if (staged) return (int)s_e[i];
            const int e = a.idx[i];
            return e >= 0 && e < a.E ? e : -1;
        };
        for (int i = tid; i < n; i += kFewThreads) {
            const int r = i / a.k, e = expert(i);
            if (e < 0) continue;
            bool first_mention = true;
            for (int t = r * a.k; t < i; ++t) first_mention &= expert(t) != e;
            if (!first_mention) continue;
            float w = staged ? s_w[i] : a.w[i];
            for (int t = i + 1; t < r * a.k + a.k; ++t)
                if (expert(t) == e) w += staged ? s_w[t] : a.w[t];
            l.gate[l.off[e] + __popcll(l.mask[e] & ((1ull << r) - 1))] = w;
        }
    }
    __syncthreads();
}

// Waits for this wave's LDS traffic and for the other waves, not for loads in flight.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, bool W8>
__device__ __forceinline__ uint32_t weight_lane(int l16, int lq) {
    return W8 ? (uint32_t)(lq * 256 + l16 * 16) : (uint32_t)(l16 * 64 + lq * 16);
}

// Steps of 16 J rows in flight, as many as registers hold (of four: two made a step of the second kernel 2,200
// cycles long, an L2 read and a half).
template <bool W8, int J, bool kDown>
constexpr int rows_ahead() { return W8 ? (J == 1 ? 4 : J == 2 ? 2 : 1) : J < 4 || kDown ? 4 : 2; }

// S waves share a unit (16 hidden units of one expert: 16 gate and 16 up rows), each its own
// share of the steps: as many small units as there are feed all CUs from the first load on, with no tile of rows to
// wait for.  Bound by the weights' bytes: 134 MB for 48 rows, 1,024 x 2,048, 16 experts in f16 take 29.2 us (4.6 TB/s) where each
// call has another layer, 24.9 where the same one again finds a part of them in the last-level cache; the 50 MB of one
// row's 8 experts, 2,048 x 768, 15.2 us (3.3 TB/s) and 13.6; 134 MB of 16 rows, 8 experts in f32 40 us and 34.  With 8-bit
// weights and more than 32 rows 4 to 10 vector and 78 scalar registers are spilled: 64 rows, 64 experts of 2,048 x 768 46 us.
template <typename T, bool W8, int NT, int S, int P>
__global__ __launch_bounds__(kFewThreads) void few_up_kernel(FewArgs a) {
    typedef Step<T, W8> St;
    constexpr int GP = kFewWaves / S;  // units a block has at a time
    extern __shared__ __align__(16) uint8_t s_dyn[];
    __shared__ f32x4_t s_part[S > 1 ? kFewWaves : 1][2][NT][kWave];
    const int places = a.rows * (a.k + a.Ecols - a.E);
    const Lists l(s_dyn, a.Ecols, places);
    if (NT == 1 && a.choice != kChoiceMade) {
        double* s_logit = reinterpret_cast<double*>(s_dyn + Lists::bytes(a.Ecols, places, false));
        if (a.choice == kChoiceOfLogits) {
            for (int i = threadIdx.x; i < a.rows * a.E; i += kFewThreads)
                s_logit[i] = a.logits[i / a.E * kMaxExperts + i % a.E];
        } else {
            const double v = logit_tile<T>(a, 0, 0, s_logit + a.rows * a.E);
            const int r = threadIdx.x / 16, e = threadIdx.x % 16;
            if (r < a.rows && e < a.E) s_logit[r * a.E + e] = v;
        }
        make_lists<false>(a, l, s_logit);  // (a barrier first)
        if (blockIdx.x == 0 && (int)threadIdx.x < a.Ecols) a.out_count[threadIdx.x] = __popcll(l.mask[threadIdx.x]);
    } else {
        make_lists<false>(a, l);
    }

    // The second kernel's counts.  Each kernel clears the other's: what a call finds does not depend on how the
    // one before it ended.
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.tile_cap; i += kFewThreads)
            __hip_atomic_store(&a.arrived[i], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = wave / S, part = wave % S;
    const int tiles = (a.H + 15) / 16, units = __builtin_amdgcn_readfirstlane(l.info[0]) * tiles;
    const int steps = (a.D + St::KS - 1) / St::KS, s0 = steps * part / S, s1 = steps * (part + 1) / S;
    const uint32_t wl = weight_lane<T, W8>(l16, lq);
    const int64_t kstep = (int64_t)a.N1 * kKBlockBytes;

    // rows through a range check: columns past D are at an offset that reads as zeros
    const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.x), 0, (int)((uint32_t)a.rows * a.D * sizeof(T)),
                                                      0x00020000);
    struct Weights {
        u32x4_t w[2][2];
        float s[2];
    };
    for (int u0 = blockIdx.x * GP; u0 < units; u0 += gridDim.x * GP) {
        const bool has = u0 + g < units;
        const int u = min(u0 + g, units - 1), li = u / tiles, ht = u - li * tiles;
        const int e = __builtin_amdgcn_readfirstlane(l.live[li]), off = __builtin_amdgcn_readfirstlane(l.off[e]);
        const int n = __builtin_amdgcn_readfirstlane(__popcll(l.mask[e]));
        const int n0 = ht / 2 * 64 + ht % 2 * 16;  // the gate rows' place; the up rows' is 32 further
        const float* b = a.b1 + (int64_t)e * a.N1 + n0 + 4 * lq;
        const float4 bg = *reinterpret_cast<const float4*>(b), bu = *reinterpret_cast<const float4*>(b + 32);
        const uint8_t* w = static_cast<const uint8_t*>(a.w1) + (int64_t)e * a.w1_expert + (int64_t)n0 * kKBlockBytes;
        const float* sg = W8 ? a.s1 + ((int64_t)e * 2 * a.hb + ht / 8) * a.kb1 : nullptr;
        const float* su = W8 ? sg + (int64_t)a.hb * a.kb1 : nullptr;
        uint32_t xo[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) xo[j] = (uint32_t)l.row[off + min(j * 16 + l16, n - 1)] * (uint32_t)(a.D * sizeof(T));
        auto fetch_w = [&](int st, Weights& d) {
            const uint8_t* p = w + 2 * st * kstep;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 2; ++q) d.w[i][q] = load16u(p + q * kstep + i * 32 * kKBlockBytes + wl);
            d.s[0] = W8 ? sg[st] : a.w1_down;
            d.s[1] = W8 ? su[st] : a.w1_down;
        };
        f32x4_t acc[2][NT];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        auto fetch_x = [&](int j, int st, u32x4_t (&d)[St::XL]) {
#pragma unroll
            for (int q = 0; q < St::XL; ++q) {
                const int k = st * St::KS + St::xk(q, lq);
                d[q] = __builtin_bit_cast(
                    u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                 rx, k < a.D ? xo[j] + (uint32_t)(k * sizeof(T)) : 0xfffffff0u, 0, 0));
            }
        };
        // 8-bit weights in code of so many row groups, as a step's values are widened once for all of them (64
        // rows, 2,048 x 768, 8 of 64 experts: 100 -> 91 us a call).  Others in one: with code for each
        // number the first kernel of 48 rows, 1,024 x 2,048, 2 of 16 experts took 37 us for 30, and loops without
        // branches, which never wait for more than the loads they need, 41.
        if constexpr (W8) {
            if (has)
                for_rows<NT>(n, [&](auto jj) {
                    constexpr int J = decltype(jj)::value, XP = rows_ahead<W8, J, false>();
                    Weights wd[P];
                    Rows<T, W8, J> xd[XP];
#pragma unroll
                    for (int p = 0; p < P; ++p)
                        if (s0 + p < s1) fetch_w(s0 + p, wd[p]);
#pragma unroll
                    for (int p = 0; p < XP; ++p)
                        if (s0 + p < s1)
#pragma unroll
                            for (int j = 0; j < J; ++j) fetch_x(j, s0 + p, xd[p].x[j]);
                    for (int st = s0; st < s1; st += P) {
#pragma unroll
                        for (int p = 0; p < P; ++p) {
                            if (st + p >= s1) break;
#pragma unroll
                            for (int c = 0; c < 2; ++c) multiply<T, W8, J>(acc[c], wd[p].w[c], xd[p % XP].x, wd[p].s[c]);
                            if (st + p + P < s1) fetch_w(st + p + P, wd[p]);
                            if (st + p + XP < s1)
#pragma unroll
                                for (int j = 0; j < J; ++j) fetch_x(j, st + p + XP, xd[p % XP].x[j]);
                        }
                    }
                });
        } else if (has) {
            constexpr int XP = rows_ahead<W8, NT, false>();
            Weights wd[P];
            Rows<T, W8, NT> xd[XP];
            auto fetch_rows = [&](int st, Rows<T, W8, NT>& d) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (j * 16 >= n) break;
                    fetch_x(j, st, d.x[j]);
                }
            };
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (s0 + p < s1) fetch_w(s0 + p, wd[p]);
#pragma unroll
            for (int p = 0; p < XP; ++p)
                if (s0 + p < s1) fetch_rows(s0 + p, xd[p]);
            for (int st = s0; st < s1; st += P) {
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    if (st + p >= s1) break;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        if (j * 16 >= n) break;
#pragma unroll
                        for (int c = 0; c < 2; ++c) multiply<T, W8, 1>(acc[c] + j, wd[p].w[c], xd[p % XP].x + j, wd[p].s[c]);
                    }
                    if (st + p + P < s1) fetch_w(st + p + P, wd[p]);
                    if (st + p + XP < s1) fetch_rows(st + p + XP, xd[p % XP]);
                }
            }
        }
        // lane (l16, lq): token row j * 16 + l16, hidden units 4 lq + (0..3) of the tile
        const int hc = ht * 16 + 4 * lq;
        auto finish = [&](int j, const f32x4_t& gv, const f32x4_t& uv) {
            const int m = j * 16 + l16;
            if (m >= n) return;
            const float fg[4] = {bg.x, bg.y, bg.z, bg.w}, fu[4] = {bu.x, bu.y, bu.z, bu.w};
            T o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                o[r] = Elt<T>::from_f32(hc + r < a.H ? swiglu<T>(gv[r] + fg[r], uv[r] + fu[r]) : 0.0f);
            typedef typename std::conditional<sizeof(T) == 2, uint2, uint4>::type Raw4;
            Raw4 raw;
            __builtin_memcpy(&raw, o, sizeof(raw));
            *reinterpret_cast<Raw4*>(static_cast<T*>(a.h) + (int64_t)(off + m) * a.ldh + hc) = raw;
        };
        if constexpr (S == 1) {
            if (has)
#pragma unroll
                for (int j = 0; j < NT; ++j) finish(j, acc[0][j], acc[1][j]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) s_part[wave][i][j][lane] = acc[i][j];
            lds_barrier();
            if (has)
                for (int j = part; j < NT; j += S) {
                    f32x4_t gv = s_part[g * S][0][j][lane], uv = s_part[g * S][1][j][lane];
#pragma unroll
                    for (int i = 1; i < S; ++i) {
                        gv += s_part[g * S + i][0][j][lane];
                        uv += s_part[g * S + i][1][j][lane];
                    }
                    finish(j, gv, uv);
                }
            lds_barrier();
        }
    }
}

// A block has 16 columns of y, or with parts > 1 a share of their sums' steps: all experts of a row end in one
// block (or kFewParts), so nothing is written between.  67 MB for 48 rows, 1,024 x 2,048, 16 experts in f16: 18.0 us (3.7
// TB/s; 64 tiles of 16 columns in 4 parts, a block a CU); 25 MB of one row's 8 experts, 2,048 x 768: 10.4 us (both from HBM: each
// call another layer).
template <typename T, bool W8, int NT, int P>
__global__ __launch_bounds__(kFewThreads) void few_down_kernel(FewArgs a) {
    typedef Step<T, W8> St;
    extern __shared__ __align__(16) uint8_t s_dyn[];
    __shared__ f32x4_t s_y[kFewWaves][16 * NT][4];  // [wave][row][4 columns each]
    __shared__ int s_last;
    const int slots = a.k + a.Ecols - a.E;
    const Lists l(s_dyn, a.Ecols, a.rows * slots);
    make_lists<true>(a, l);
    if (blockIdx.x == 0 && threadIdx.x < kFewGroups)  // the router's kernel's counts
        __hip_atomic_store(&a.arrived[a.tile_cap + threadIdx.x], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tile = blockIdx.x / a.parts, part = blockIdx.x % a.parts, n0 = tile * 16;
    const int steps = (a.H + St::KS - 1) / St::KS;  // of an expert
    const int chosen = __builtin_amdgcn_readfirstlane(l.info[0]), total = chosen * steps, shares = a.parts * kFewWaves;
    const int share = part * kFewWaves + wave;
    const int s0 = (int)((int64_t)total * share / shares), s1 = (int)((int64_t)total * (share + 1) / shares);
    const uint32_t wl = weight_lane<T, W8>(l16, lq);
    const int64_t kstep = (int64_t)a.N2 * kKBlockBytes;
    const int live_h = (a.H + 15) / 16 * 16;  // columns of h that are written

    for (int r = lane; r < 16 * NT * 4; r += kWave) s_y[wave][r / 4][r % 4] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    struct At {
        int li, st, e, off, n;  // a chosen expert and a step of it
    };
    auto place = [&](At& t) {
        t.e = __builtin_amdgcn_readfirstlane(l.live[t.li]);
        t.off = __builtin_amdgcn_readfirstlane(l.off[t.e]);
        t.n = __builtin_amdgcn_readfirstlane(__popcll(l.mask[t.e]));
    };
    // to the step after: past an expert's last one the next expert's
    auto next = [&](At& t) {
        if (++t.st < steps) return;
        t.st = 0;
        t.li = min(t.li + 1, chosen - 1);
        place(t);
    };
    struct Weights {
        u32x4_t w[2];
        float s;
    };
    const auto rh = __builtin_amdgcn_make_buffer_rsrc(a.h, 0, (int)((uint32_t)(a.rows * slots) * (uint32_t)(a.ldh * sizeof(T))),
                                                      0x00020000);
    auto fetch_w = [&](At& t, Weights& d) {
        const uint8_t* p = static_cast<const uint8_t*>(a.w2) + (int64_t)t.e * a.w2_expert + (int64_t)n0 * kKBlockBytes +
                           2 * t.st * kstep;
#pragma unroll
        for (int q = 0; q < 2; ++q) d.w[q] = load16u(p + q * kstep + wl);
        d.s = W8 ? a.s2[((int64_t)t.e * a.nb2 + n0 / kFp8Block) * a.kb2 + t.st] : a.w2_down;
        next(t);
    };
    f32x4_t acc[NT];
    auto clear = [&] {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    };
    float4 b2;  // the lane's biases of the expert at hand
    auto biases = [&](const At& t) { b2 = *reinterpret_cast<const float4*>(a.b2 + (int64_t)t.e * a.N2 + n0 + 4 * lq); };
    // the sums of an expert so far, weighed, to the rows' (each row of it is one lane's)
    auto flush = [&](const At& t, bool bias) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int m = j * 16 + l16;
            if (m < t.n) {
                const float w = l.gate[t.off + m];
                f32x4_t v = acc[j];
                if (bias) v += f32x4_t{b2.x, b2.y, b2.z, b2.w};
                f32x4_t& to = s_y[wave][l.row[t.off + m]][lq];
#pragma unroll
                for (int r = 0; r < 4; ++r) to[r] = __builtin_fmaf(v[r], w, to[r]);
            }
        }
        clear();
    };
    clear();
    if (s0 < s1) {
        At at = {s0 / steps, s0 % steps, 0, 0, 0};
        int most = 0;  // rows of an expert of this wave's
        for (int li = at.li; li <= (s1 - 1) / steps; ++li)
            most = max(most, __builtin_amdgcn_readfirstlane(__popcll(l.mask[l.live[li]])));
        place(at);
        bool whole = at.st == 0;  // the expert's first step is this wave's
        biases(at);
        for_rows<NT>(most, [&](auto jj) {
            constexpr int J = decltype(jj)::value, XP = rows_ahead<W8, J, true>();
            auto fetch_x = [&](At& t, Rows<T, W8, J>& d) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (J > 1 && j * 16 >= t.n) break;
                    const uint32_t h = (uint32_t)(t.off + min(j * 16 + l16, t.n - 1)) * (uint32_t)(a.ldh * sizeof(T));
#pragma unroll
                    for (int q = 0; q < St::XL; ++q) {
                        const int k = t.st * St::KS + St::xk(q, lq);
                        d.x[j][q] = __builtin_bit_cast(
                            u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                         rh, k < live_h ? h + (uint32_t)(k * sizeof(T)) : 0xfffffff0u, 0, 0));
                    }
                }
                next(t);
            };
            At aw = at, ax = at;  // of the weights' and the rows' loads
            Weights wd[P];
            Rows<T, W8, J> xd[XP];
#pragma unroll
            for (int p = 0; p < XP; ++p)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int q = 0; q < St::XL; ++q) xd[p].x[j][q] = u32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (s0 + p < s1) fetch_w(aw, wd[p]);
#pragma unroll
            for (int p = 0; p < XP; ++p)
                if (s0 + p < s1) fetch_x(ax, xd[p]);
            for (int s = s0; s < s1; s += P) {
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    if (s + p >= s1) break;
                    if (at.st == steps) {
                        flush(at, whole);
                        ++at.li;
                        at.st = 0;
                        place(at);
                        biases(at);
                        whole = true;
                    }
                    multiply<T, W8, J>(acc, wd[p].w, xd[p % XP].x, wd[p].s);  // (rows past the expert's: not used)
                    ++at.st;
                    if (s + p + P < s1) fetch_w(aw, wd[p]);
                    if (s + p + XP < s1) fetch_x(ax, xd[p % XP]);
                }
            }
        });
        flush(at, whole);
    }
    __syncthreads();
    // the waves' sums in wave order; thread (row, column quarter)
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    const int row = tid / 4, c = tid % 4;
    static_assert(kFewThreads >= 64 * 4, "a thread for 4 columns of each row");
    if (row < a.rows) {
        v = s_y[0][row][c];
#pragma unroll
        for (int w = 1; w < kFewWaves; ++w) v += s_y[w][row][c];
    }
    if (a.parts > 1) {
        // The last block to arrive adds the shares, in their order.  Blocks of a tile run on
        // different XCDs, whose L2 caches are not coherent: the shares are written and read past
        // them (agent-scope cache policy), and written, as the wait says, before the block is
        // counted.  So nothing has to be written back or thrown away: a release and an acquire
        // around the count took 3 us, fences of every wave 50.
        constexpr int kSc1 = 16;
        const auto rs = __builtin_amdgcn_make_buffer_rsrc(a.partial + (int64_t)tile * kFewParts * kFewRows * 16, 0,
                                                          kFewParts * kFewRows * 64, 0x00020000);
        if (row < a.rows)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), rs, (part * kFewRows + row) * 64 + c * 16, 0,
                                                   kSc1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0)
            s_last = __hip_atomic_fetch_add(&a.arrived[tile], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.parts - 1;
        __syncthreads();
        if (!s_last) return;
        if (row < a.rows) {
            f32x4_t t[kFewParts];
#pragma unroll
            for (int p = 0; p < kFewParts; ++p)  // (past the last part: any of them, not used)
                t[p] = __builtin_bit_cast(
                    f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (min(p, a.parts - 1) * kFewRows + row) * 64 + c * 16, 0, kSc1));
            v = t[0];
#pragma unroll
            for (int p = 1; p < kFewParts; ++p)
                if (p < a.parts) v += t[p];
        }
    }
    const int col = n0 + 4 * c;
    if (row < a.rows && col < a.D) {  // (D % 8 == 0: four columns are real or padding)
        T o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = Elt<T>::from_f32(v[r]);
        typedef typename std::conditional<sizeof(T) == 2, uint2, uint4>::type Raw4;
        Raw4 raw;
        __builtin_memcpy(&raw, o, sizeof(raw));
        *reinterpret_cast<Raw4*>(static_cast<T*>(a.y) + (int64_t)row * a.D + col) = raw;
    }
}

// The lists are dynamic LDS; more than 64 KB in a block has to be asked for.
template <typename F>
hipError_t launch(F kernel, int64_t grid, size_t fixed, size_t lds, const FewArgs& a, hipStream_t s) {
    if (fixed + lds > 160 * 1024) return hipErrorInvalidValue;
    if (fixed + lds > 64 * 1024) {
        const hipError_t e =
            hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    launch_kernel(kernel, dim3((unsigned)grid), dim3(kFewThreads), (uint32_t)lds, s, a);
    return hipGetLastError();
}

template <typename T, bool W8, int NT>
hipError_t launch_nt(FewArgs a, hipStream_t s) {
    constexpr int P = 4;  // steps of weights in flight
    typedef Step<T, W8> St;
    const int slots = a.k + a.Ecols - a.E, places = a.rows * slots;
    const int tiles = (a.H + 15) / 16, live = std::min(a.E, a.rows * a.k) + a.Ecols - a.E;
    const int64_t units = (int64_t)tiles * live;
    const size_t lds1 = Lists::bytes(a.Ecols, places, false) + (a.choice != kChoiceMade ? (size_t)a.rows * a.E * 8 : 0) +
                        (a.choice == kChoiceOfRows ? (size_t)kFewWaves * 256 * 8 : 0),
                 lds2 = Lists::bytes(a.Ecols, places, true);
    // The share of a unit's steps that a wave takes (1 / S) by the steps that the longest wave then walks, one block of
    // eight waves a CU, a round's first loads as long as six steps; of equal ones the fewest waves a unit, which have the
    // fewest sums to exchange.
    const int steps = (a.D + St::KS - 1) / St::KS;
    int S = 1;
    int64_t least = INT64_MAX;
    for (const int c : {1, 2, 4, 8}) {
        const int64_t rounds = (units * c + 256 * kFewWaves - 1) / (256 * kFewWaves), walk = rounds * (6 + (steps + c - 1) / c);
        if (walk < least) {
            least = walk;
            S = c;
        }
    }
    const int64_t grid = std::min<int64_t>((units * S + kFewWaves - 1) / kFewWaves, 256);
    constexpr size_t fixed1 = kFewWaves * (2 * NT * kWave * 16 + 256) + 64, fixed2 = kFewWaves * NT * kWave * 16 + kStaged * 6 + 64;
    hipError_t e = S == 1   ? launch(few_up_kernel<T, W8, NT, 1, P>, grid, fixed1, lds1, a, s)
                   : S == 2 ? launch(few_up_kernel<T, W8, NT, 2, P>, grid, fixed1, lds1, a, s)
                   : S == 4 ? launch(few_up_kernel<T, W8, NT, 4, P>, grid, fixed1, lds1, a, s)
                            : launch(few_up_kernel<T, W8, NT, 8, P>, grid, fixed1, lds1, a, s);
    if (e != hipSuccess) return e;
    const int ntiles = (a.D + 15) / 16;
    // (no part of a tile without work for all of its waves)
    a.parts = std::max(1, std::min({kFewParts, 256 / ntiles, live * ((a.H + St::KS - 1) / St::KS) / (kFewWaves * 4)}));
    return launch(few_down_kernel<T, W8, NT, P>, ntiles * a.parts, fixed2, lds2, a, s);
}

template <typename T>
hipError_t launch_route(const FewArgs& a, hipStream_t s) {
    const size_t lds = (size_t)16 * a.E * sizeof(double);  // (at most 32 KB beside 17 KB)
    launch_kernel(few_route_kernel<T>, dim3((unsigned)(a.E + 15) / 16, (unsigned)(a.rows + 15) / 16), dim3(kFewThreads),
                  (uint32_t)lds, s, a);
    return hipGetLastError();
}

template <typename T, bool W8>
hipError_t launch_few_t(FewArgs a, hipStream_t s) {
    // Who chooses.  Up to 16 rows: every block of the first kernel, from logits that it makes itself
    // where the router's weights and the rows are a few KB, else from those of a kernel that has a
    // block for 16 experts.  More rows: that kernel's last blocks.  (Two rows of 64, 4 experts: 21
    // us a call with a kernel for the router, 18 without; one row of 2,048, 64 experts: the router's
    // kernel 10 us with the choice, 4.6 without.)
    a.choice = kChoiceMade;
    if (a.wr && a.rows <= 16)
        a.choice = a.E <= 16 && (int64_t)(a.rows + a.E) * a.D * (int)sizeof(T) <= 64 * 1024 ? kChoiceOfRows : kChoiceOfLogits;
    if (a.wr && a.choice != kChoiceOfRows) {
        const hipError_t e = launch_route<T>(a, s);
        if (e != hipSuccess) return e;
    }
    if (a.rows <= 16) return launch_nt<T, W8, 1>(a, s);
    if (a.rows <= 32) return launch_nt<T, W8, 2>(a, s);
    return launch_nt<T, W8, 4>(a, s);
}

}  // namespace

hipError_t launch_few(DType dt, const FewArgs& a, hipStream_t s) {
    if (a.rows < 1 || a.rows > kFewRows || a.D < 8 || a.D % 8 != 0 || a.E < 1 || a.E > kMaxExperts || a.k < 1 ||
        a.k > a.Ecols || (int64_t)a.rows * a.D > (1 << 28) || (int64_t)a.rows * (a.k + 1) * a.ldh > (1 << 28) ||
        (a.D + 15) / 16 > a.tile_cap)
        return hipErrorInvalidValue;
    const bool w8 = a.s1 != nullptr;
    switch (dt) {
        case DType::F32: return w8 ? hipErrorInvalidValue : launch_few_t<float, false>(a, s);
        case DType::BF16: return w8 ? launch_few_t<__bf16, true>(a, s) : launch_few_t<__bf16, false>(a, s);
        case DType::F16: return w8 ? launch_few_t<_Float16, true>(a, s) : launch_few_t<_Float16, false>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace nomas
