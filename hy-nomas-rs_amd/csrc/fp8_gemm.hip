// Products of 8-bit matrices with a scale for each block of 128:
//   y[m, n] = sum over blocks kb of sa[m, kb] sb[n / 128, kb] (sum over k of the block a[m, k] b[n, k]) + bias[n]
//
// One v_mfma_f32_16x16x128_f8f6f4 makes a block's sums for 16 x 16 outputs; they are scaled and
// added by the vector units, four fused multiply-adds a lane.  The weights are the first
// operand: a lane then holds four neighbouring outputs of one row, whose scale is one register.
//
// The 8-bit matrix instructions do not add in f32 throughout: of each 8 products (neighbours
// in k) they keep the bits down to 2^-13 of the largest one's power of two, and add those sums in f32
// (measured: 2^16 + 2^3 is exact, 2^16 + 2^2 is not; the 16x16x32 form does the same).  On random
// values that is 1.4e-5 of the result, at most 8.5e-4 of the terms' magnitudes: far below a 16-bit
// result's own rounding, but not an f32 result's.  Those are made with bf16 MFMAs
// from the same bytes (every e4m3 is a bf16): exact products, f32 sums, half the rate.
#include "fp8.hpp"
#include "lds_dma.hpp"
#include "mfma.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace nomas {

namespace {

__device__ __forceinline__ f32x4_t mfma_fp8(const i32x8_t& a, const i32x8_t& b) {
    const f32x4_t z = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, z, 0, 0, 0, 0, 0, 0);
}
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// The lane's 32 values of a fragment, for 16-bit results as they are, for f32 ones widened.
template <bool kExact> struct Frag;
template <> struct Frag<false> {
    i32x8_t v;
    __device__ __forceinline__ void set(const i32x8_t& b) { v = b; }
};
template <> struct Frag<true> {
    bf16x8_t v[4];
    __device__ __forceinline__ void set(const i32x8_t& b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[i], 1.0f, false);
            const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[i], 1.0f, true);
            v[i / 2][i % 2 * 4] = lo[0];
            v[i / 2][i % 2 * 4 + 1] = lo[1];
            v[i / 2][i % 2 * 4 + 2] = hi[0];
            v[i / 2][i % 2 * 4 + 3] = hi[1];
        }
    }
};
__device__ __forceinline__ f32x4_t dot(const Frag<false>& a, const Frag<false>& b) { return mfma_fp8(a.v, b.v); }
__device__ __forceinline__ f32x4_t dot(const Frag<true>& a, const Frag<true>& b) {
    f32x4_t c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}
template <typename T> using FragOf = Frag<sizeof(T) == 4>;
__device__ __forceinline__ i32x8_t join(const i32x4_t& lo, const i32x4_t& hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Four neighbouring outputs of a row.
template <typename T>
__device__ __forceinline__ void put4(T* row, int n, int N, const f32x4_t& v, bool whole) {
    T o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = Elt<T>::from_f32(v[r]);
    if (whole && n + 4 <= N) {
        typedef typename std::conditional<sizeof(T) == 2, uint2, uint4>::type Raw4;
        Raw4 raw;
        __builtin_memcpy(&raw, o, sizeof(raw));
        *reinterpret_cast<Raw4*>(row + n) = raw;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < N) row[n + r] = o[r];
    }
}

// What is made of the products:
//  kStore  y (M x N) in T, with a bias
//  kGlu    the hidden activations of a SwiGLU feed-forward: b's rows are its packed gate and up rows
//          (32 of the one, 32 of the other), scales for squares of 128 gate rows, then of the up
//          rows; silu(gate + bias) (up + bias) in f32 as 8-bit values with a scale for each
//          128 of them (tile kernel: a tile has whole blocks) or as they are (few rows)
enum { kStore = 0, kGlu = 1 };

// ---- the scales' product ---------------------------------------------------------
// sa sb leaves f32's range where the results do not: two of 2^-70 beside sums of 2^20, two of 2^70 beside sums
// of 2^-14, or beside a sum of 0.  So the sums are taken times 2^32.  Products of scales down to 2^-158 are
// then normal numbers, and the bits that smaller ones lose are below 2^-156 of a result: under 1/64 of f32's
// last bit.  Products from 2^55 on (a row's sum can add 2^40 of one) and infinities are seen by a compare a
// step; a wave that saw one makes its sums again, with the scales' powers of two apart.  (NaN needs no second try.)
constexpr float kScaleUp = 0x1p32f, kScaleDown = 0x1p-32f, kScaleMost = 0x1p87f;
__device__ __forceinline__ bool too_large(float s) { return __builtin_fabsf(s) >= kScaleMost; }

// The wave's sums over blocks kt0, kt0 + step, ... for any scales, to put(i, j, sums): a block's sum times the scales'
// mantissas, then their powers of two in one step.  w, x: the wave's first rows; rows past last_n, last_m (the
// matrices' last ones, as seen from there) are the last one again.  bs: the scales of its weights' block, with kGlu of
// the gate rows, the up rows' `up` further.  One fragment at a time from global memory, to keep out of the other
// path's registers: 1,111 x 2,667 x 1,008 in bf16 59 us for 18, 14,232 x 8,192 x 2,048 4,180 for 280.
template <typename T, int MODE, int NI, int NJ, typename F>
__device__ __forceinline__ void sum_any_scales(const Fp8GemmArgs& a, const uint8_t* w, const uint8_t* x, const float* as,
                                               const float* bs, int64_t up, int last_n, int last_m, int kt0, int step, F put) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
    const int kb = (a.K + kFp8Block - 1) / kFp8Block;
    auto frag = [&](const uint8_t* p, int k) {
        const i32x4_t z = {0, 0, 0, 0};
        FragOf<T> f;
        f.set(join(k < a.K ? *reinterpret_cast<const i32x4_t*>(p + k) : z,
                   k + 16 < a.K ? *reinterpret_cast<const i32x4_t*>(p + k + 16) : z));
        return f;
    };
#pragma unroll 1
    for (int i = 0; i < NI; ++i) {
        const uint8_t* wi = w + (int64_t)min(i * 16 + l16, last_n) * a.K;
        const float* sbs = bs + (MODE == kGlu && i % 4 >= 2 ? up : 0);
#pragma unroll 1
        for (int j = 0; j < NJ; ++j) {
            const int m = min(j * 16 + l16, last_m);
            const uint8_t* xj = x + (int64_t)m * a.K;
            f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int kt = kt0; kt < kb; kt += step) {
                const int k = kt * kFp8Block + lq * 32;
                const f32x4_t t = dot(frag(wi, k), frag(xj, k));
                const float sa = as[(int64_t)m * kb + kt], sb = sbs[kt];
                const float f = __builtin_amdgcn_frexp_mantf(sa) * __builtin_amdgcn_frexp_mantf(sb);
                const int e = __builtin_amdgcn_frexp_expf(sa) + __builtin_amdgcn_frexp_expf(sb);
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[r] += __builtin_ldexpf(t[r] * f, e);
            }
            put(i, j, sum);
        }
    }
}

// ---- tiles through LDS ---------------------------------------------------------
// A block's WN x WM waves share a tile of 16 NI WN weight rows and 16 NJ WM rows;
// K-blocks of 128 bytes a row go through a ring of two LDS stages, filled by direct loads of
// whole 128-byte rows.  16-byte chunk c of row r is kept at chunk c ^ (r % 8), so that the
// fragment reads (one chunk of 8 rows at a time) touch every bank once.  Bound by the matrix pipes and the scaling's
// vector instructions beside them: 14,232 x 8,192 x 2,048 in bf16 245-280 us by the card's clock (1,710-1,950 TFLOP/s; the pipes
// are busy 41% of the cycles); the rest of a tile's time is its first loads and its outputs.  f32 results 487 us.  Where there is less
// than a round of tiles, a step waits for its loads (0.8 us; f32 1.2): 1,111 x 2,667 x 1,008 in f16, 189 tiles of 128 x 128, takes
// 16.5 us, and 13.4 with 2,672 columns, whose outputs leave in whole lines.
template <typename T, int MODE, int NI, int NJ, int WN, int WM>
__global__ __launch_bounds__(WN * WM * kWave) void fp8_tile_kernel(Fp8GemmArgs a, int tiles_m, int tiles_n) {
    constexpr int NW = WN * WM, BN = 16 * NI * WN, BM = 16 * NJ * WM;
    constexpr int kStage = (BN + BM) * kFp8Block;
    __shared__ __align__(1024) uint8_t s_ring[2][kStage];
    __shared__ float s_sa[2][BM], s_sb[2][kWave];
    constexpr int QN = BN / 8 / NW, QM = BM / 8 / NW;  // loads of 8 rows a wave

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;

    // one contiguous share of the tiles per XCD (block i runs on XCD i % 8), groups of eight
    // row tiles walked column by column
    const int tiles = tiles_m * tiles_n, share = (tiles + kNumXcd - 1) / kNumXcd;
    const int u = (int)(blockIdx.x % kNumXcd) * share + (int)(blockIdx.x / kNumXcd);
    if ((int)(blockIdx.x / kNumXcd) >= share || u >= tiles) return;
    constexpr int G = 8;
    const int group = u / (G * tiles_n), first = group * G, gm = min(G, tiles_m - first);
    const int in = u - group * G * tiles_n;
    const int tm = first + in % gm, tn = in / gm;
    const int64_t m0 = (int64_t)tm * BM;
    const int n0 = tn * BN;
    const int K = a.K, kb = (K + kFp8Block - 1) / kFp8Block;
    const int rows_n = min(BN, a.N - n0), rows_m = (int)min<int64_t>(BM, a.M - m0);

    // rows past the matrix fail the range check and read as zeros
    const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.b) + (int64_t)n0 * K, 0,
                                                      (int)((uint32_t)rows_n * (uint32_t)K), 0x00020000);
    const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.a) + m0 * K, 0,
                                                      (int)((uint32_t)rows_m * (uint32_t)K), 0x00020000);
    // (the first of the wave's loads of 8 rows; the others' offsets are made where they go out: registers are short)
    const int chunk = (lane & 7) ^ (lane >> 3);
    const uint32_t v0 = (uint32_t)(lane >> 3) * (uint32_t)K + chunk * 16;
    // the scales of the rows: one per thread of the first BM / 64 waves (past the end the last row's)
    const uint32_t vs = (uint32_t)min(tid % BM, rows_m - 1) * (uint32_t)kb * 4;
    const float* as = a.as + m0 * kb;
    // ... and of the tile's weights: blocks of 128 rows, with kGlu the gate rows' and the up rows'.  (A
    // load of them to registers waited for all the direct loads issued before it.)
    static_assert(kFp8Block % (16 * NI) == 0 && BN / kFp8Block <= 2, "one weight scale a wave");
    const uint32_t vsb = MODE == kGlu ? (uint32_t)(tn + (lane & 1) * tiles_n) * (uint32_t)kb * 4
                                      : (uint32_t)min(n0 / kFp8Block + (lane & 1), (a.N - 1) / kFp8Block) * (uint32_t)kb * 4;
    const uint32_t sbs = lds_addr(&s_sb[0][0]);
    // the first waves load the rows' scales, the others the weights'
    static_assert(NW > BM / kWave, "a wave for the weights' scales");
    const bool rows_scales = wave < BM / kWave;
    const float* scales = rows_scales ? as : a.bs;
    const uint32_t scales_stage = rows_scales ? BM * 4 : kWave * 4;
    const uint32_t ring = lds_addr(&s_ring[0][0]), sas = lds_addr(&s_sa[0][0]);

    // load q of a wave for block kt: of the QN + QM tile loads, then the scales
    auto issue = [&](int kt, int q) {
        const uint32_t at = ring + (kt & 1) * kStage, k0 = (uint32_t)kt * kFp8Block;
        const bool out = (int)k0 + chunk * 16 >= K;  // (only in the last block, or past it)
        uint32_t v = v0;
        asm volatile("" : "+v"(v));  // (else all loads' offsets are kept, and registers spilled)
        if (q < QN) {
            lds_dma16_buf_s(rb, out ? 0xfffffff0u : v + (uint32_t)(wave * QN + q) * 8 * (uint32_t)K, k0,
                            at + (wave * QN + q) * 1024);
        } else if (q < QN + QM) {
            const int m = q - QN;
            lds_dma16_buf_s(ra, out ? 0xfffffff0u : v + (uint32_t)(wave * QM + m) * 8 * (uint32_t)K, k0,
                            at + (BN / 8 + wave * QM + m) * 1024);
        } else {
            // (no branch here: the compiler moved all scaling behind it)
            lds_dma4(scales + min(kt, kb - 1), rows_scales ? vs : vsb, (rows_scales ? sas + wave * 256 : sbs) + (kt & 1) * scales_stage);
        }
    };
    constexpr int kLoads = QN + QM + 1;

    f32x4_t acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    bool beyond = false;
    const int sw = l16 & 7;
    const int c0 = (2 * lq) ^ sw, c1 = (2 * lq + 1) ^ sw;

#pragma unroll
    for (int q = 0; q < kLoads; ++q) issue(0, q);
    for (int kt = 0; kt < kb; ++kt) {
        wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // stage kt has landed, and all have read the other one
        asm volatile("" ::: "memory");
        const uint8_t* wt = s_ring[kt & 1] + (wn * NI * 16 + l16) * kFp8Block;
        const uint8_t* xt = s_ring[kt & 1] + (BN + wm * NJ * 16 + l16) * kFp8Block;
        auto frag = [&](const uint8_t* p, int i) {
            return join(*reinterpret_cast<const i32x4_t*>(p + i * 16 * kFp8Block + c0 * 16),
                        *reinterpret_cast<const i32x4_t*>(p + i * 16 * kFp8Block + c1 * 16));
        };
        const float sb = s_sb[kt & 1][MODE == kGlu ? 0 : wn * 16 * NI / kFp8Block] * kScaleUp;
        const float sb2 = MODE == kGlu ? s_sb[kt & 1][1] * kScaleUp : 0.0f;
        beyond = beyond || too_large(sb) || too_large(sb2);  // (times a scale of 0: NaN)
        FragOf<T> x[NJ], w[2];
        float s[NJ], s2[NJ];
        w[0].set(frag(wt, 0));
#pragma unroll
        for (int j = 0; j < NJ; ++j) x[j].set(frag(xt, j));
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const float sa = s_sa[kt & 1][wm * NJ * 16 + j * 16 + l16];
            s[j] = sa * sb;
            s2[j] = MODE == kGlu ? sa * sb2 : 0.0f;
            beyond = beyond || too_large(s[j]) || too_large(s2[j]);
        }
        // Two products a turn; beside them the scaling of the two before, the next weights' read and a share of the
        // loads of block kt + 1: a direct load goes out every 35 cycles a CU at most, and all of them at a
        // step's start held its first products back.
        constexpr int kTurns = NI * NJ / 2, kPer = (kLoads + kTurns - 1) / kTurns;
        f32x4_t t[2][2];
        auto scale = [&](int u) {
            const int i = u / (NJ / 2);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = u % (NJ / 2) * 2 + h;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[i][j][r] = __builtin_fmaf(t[u % 2][h][r], MODE == kGlu && i % 4 >= 2 ? s2[j] : s[j], acc[i][j][r]);
            }
        };
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
            const int i = u / (NJ / 2), j = u % (NJ / 2) * 2;
            if (j == 0 && i + 1 < NI) w[(i + 1) % 2].set(frag(wt, i + 1));
            t[u % 2][0] = dot(w[i % 2], x[j]);
            t[u % 2][1] = dot(w[i % 2], x[j + 1]);
#pragma unroll
            for (int q = u * kPer; q < (u + 1) * kPer && q < kLoads; ++q) issue(kt + 1, q);  // (past the end: zeros)
            if (u > 0) scale(u - 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        scale(kTurns - 1);
    }
    wait_vmcnt<0>();  // (the loads past the end have written their zeros)
    float down = kScaleDown;
    if (__any(beyond)) {
        const int wr = n0 + wn * NI * 16;  // the wave's first weight row, and row
        const int64_t xr = m0 + wm * NJ * 16;
        const int block = MODE == kGlu ? tn : min(wr, a.N - 1) / kFp8Block;
        f32x4_t sums[NI][NJ];
        sum_any_scales<T, MODE, NI, NJ>(a, a.b + (int64_t)wr * K, a.a + xr * K, a.as + xr * kb, a.bs + (int64_t)block * kb,
                                        (int64_t)tiles_n * kb, a.N - 1 - wr, (int)min<int64_t>(a.M - 1 - xr, BM), 0, 1,
                                        [&](int i, int j, const f32x4_t& v) { sums[i][j] = v; });
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = sums[i][j];
        down = 1.0f;
    }

    if constexpr (MODE == kGlu) {
        // a lane's gate values of weight blocks i and up values of i + 2 are of the same hidden
        // units; the tile is 128 of them, a block of the output
        static_assert(MODE != kGlu || (NI == 8 && WN == 2), "a tile is 128 hidden units");
        const int H = a.N / 2, hb = H / kFp8Block;
        uint32_t top[NJ];
        int hc[4];  // the lane's four neighbouring units, four times
#pragma unroll
        for (int p = 0; p < 4; ++p) hc[p] = n0 / 2 + wn * 64 + p / 2 * 32 + p % 2 * 16 + 4 * lq;
#pragma unroll
        for (int j = 0; j < NJ; ++j) top[j] = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int i = p / 2 * 4 + p % 2, at = n0 + wn * 128 + i * 16 + 4 * lq;
            const float4 bg = *reinterpret_cast<const float4*>(a.bias + at);
            const float4 bu = *reinterpret_cast<const float4*>(a.bias + at + 32);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                acc[i][j] = acc[i][j] * down + f32x4_t{bg.x, bg.y, bg.z, bg.w};
                acc[i + 2][j] = acc[i + 2][j] * down + f32x4_t{bu.x, bu.y, bu.z, bu.w};
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float h = hc[p] + r < a.hidden ? swiglu<__bf16>(acc[i][j][r], acc[i + 2][j][r]) : 0.0f;
                    acc[i][j][r] = h;
                    top[j] = max(top[j], __float_as_uint(h) & 0x7fffffffu);
                }
            }
        }
        __syncthreads();  // (all have read the last stage)
        uint32_t* s_top = reinterpret_cast<uint32_t*>(&s_ring[0][0]);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 16));
            top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 32));
            if (lq == 0) s_top[((wm * NJ + j) * 16 + l16) * 2 + wn] = top[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int m = (wm * NJ + j) * 16 + l16;
            if (m >= rows_m) continue;
            const float s = fp8_scale(max(s_top[m * 2], s_top[m * 2 + 1]));
            const Fp8Quot d(s);
            uint8_t* q = static_cast<uint8_t*>(a.y) + (m0 + m) * H;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const f32x4_t& h = acc[p / 2 * 4 + p % 2][j];
                *reinterpret_cast<uint32_t*>(q + hc[p]) = fp8_pack4(d(h[0]), d(h[1]), d(h[2]), d(h[3]));
            }
            if (wn == 0 && lq == 0) a.y_scale[(m0 + m) * hb + tn] = s;
        }
        return;
    }
    T* y = static_cast<T*>(a.y);
    float bias[NI][4];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = n0 + (wn * NI + i) * 16 + 4 * lq + r;
            bias[i][r] = a.bias && n < a.N ? a.bias[n] : 0.0f;
        }
    constexpr int V = 16 / (int)sizeof(T), kWide = 16 * NI;  // outputs of a 16-byte store, and of a row of the wave
    if (n0 + BN <= a.N && a.N % V == 0) {
        // Sixteen rows at a time through LDS of the wave's own: a lane has four neighbouring outputs of a
        // row, and stores of those (32 bytes of each row at a time) took a third of a product of 2,048 columns.
        constexpr int kRow = kWide * (int)sizeof(T) + 16;  // (16 bytes more: rows start at other banks)
        static_assert(NW * 16 * kRow <= 2 * kStage, "in the ring");
        __syncthreads();  // (all have read the last stage)
        uint8_t* lds = &s_ring[0][0] + wave * 16 * kRow;
        constexpr int kLanesRow = kWide / V, kRowsStore = kWave / kLanesRow;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                T o[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = Elt<T>::from_f32(__builtin_fmaf(acc[i][j][r], down, bias[i][r]));
                __builtin_memcpy(lds + l16 * kRow + (i * 16 + 4 * lq) * sizeof(T), o, sizeof(o));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (one wave: nothing else to wait for)
#pragma unroll
            for (int q = 0; q < 16 / kRowsStore; ++q) {
                const int row = q * kRowsStore + lane / kLanesRow, c = lane % kLanesRow;
                const u32x4_t v = *reinterpret_cast<const u32x4_t*>(lds + row * kRow + c * 16);
                const int m = (wm * NJ + j) * 16 + row;
                if (m < rows_m) *reinterpret_cast<u32x4_t*>(y + (m0 + m) * a.N + n0 + wn * kWide + c * V) = v;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        return;
    }
    const bool whole = a.N % 4 == 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int n = n0 + (wn * NI + i) * 16 + 4 * lq;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int m = (wm * NJ + j) * 16 + l16;
            f32x4_t v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = __builtin_fmaf(acc[i][j][r], down, bias[i][r]);
            if (m < rows_m) put4(y + (m0 + m) * a.N, n, a.N, v, whole);
        }
    }
}

// ---- few rows --------------------------------------------------------------------
// 16 NT rows x 16 NI weight rows a block; its NW waves take the K-blocks in turn, operands
// straight from global memory, and add their sums in LDS in wave order: LDS holds nothing that two waves
// read, and every CU has loads under way at once.  Bound by latency: 16.8 MB of one row's 8,192 x 2,048 take 5 us, 40
// rows of 1,536 x 4,096 in f32 12.4 (96 blocks, each of them all of K).  The gate and up kernel of 17 to 32 rows spills 9 registers.
template <typename T, int MODE, int NI, int NT, int NW, int P>
__global__ __launch_bounds__(NW * kWave) void fp8_rows_kernel(Fp8GemmArgs a) {
    constexpr int BN = 16 * NI, BM = 16 * NT;
    __shared__ f32x4_t s_part[NW][NI][NT][kWave];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * BN;
    const int64_t m0 = (int64_t)blockIdx.y * BM;
    const int K = a.K, kb = (K + kFp8Block - 1) / kFp8Block;
    const int rows_m = (int)min<int64_t>(BM, a.M - m0);
    const uint8_t* bt = a.b + (int64_t)n0 * K;
    const uint8_t* at = a.a + m0 * K;
    const float* as = a.as + m0 * kb;
    // (rows past the matrices: the last one again, never stored)
    int64_t wo[NI], xo[NT];
#pragma unroll
    for (int i = 0; i < NI; ++i) wo[i] = (int64_t)min(i * 16 + l16, a.N - 1 - n0) * K + lq * 32;
#pragma unroll
    for (int j = 0; j < NT; ++j) xo[j] = (int64_t)min(j * 16 + l16, rows_m - 1) * K + lq * 32;

    struct Step {
        i32x4_t w[NI][2], x[NT][2];
        float sa[NT], sb, sb2;
    };
    const int hb = a.N / 2 / kFp8Block;  // (kGlu)
    const float* bs = a.bs + (int64_t)(MODE == kGlu ? n0 / 2 / kFp8Block : n0 / kFp8Block) * kb;
    auto load = [&](int kt, Step& s) {
        const int k = kt * kFp8Block + lq * 32;
        const bool ok0 = k < K, ok1 = k + 16 < K;  // (false in the last block only)
        const i32x4_t z = {0, 0, 0, 0};
        const int64_t o = (int64_t)kt * kFp8Block;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const uint8_t* p = bt + wo[i] + o;
            s.w[i][0] = ok0 ? *reinterpret_cast<const i32x4_t*>(p) : z;
            s.w[i][1] = ok1 ? *reinterpret_cast<const i32x4_t*>(p + 16) : z;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint8_t* p = at + xo[j] + o;
            s.x[j][0] = ok0 ? *reinterpret_cast<const i32x4_t*>(p) : z;
            s.x[j][1] = ok1 ? *reinterpret_cast<const i32x4_t*>(p + 16) : z;
            s.sa[j] = as[(int64_t)min(j * 16 + l16, rows_m - 1) * kb + kt];
        }
        s.sb = bs[kt];
        s.sb2 = MODE == kGlu ? bs[(int64_t)hb * kb + kt] : 0.0f;
    };
    static_assert(kFp8Block % BN == 0, "one weight scale a block");
    f32x4_t acc[NI][NT];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    bool beyond = false;
    Step st[P];
#pragma unroll
    for (int p = 0; p < P; ++p)
        if (wave + p * NW < kb) load(wave + p * NW, st[p]);
    for (int k0 = wave; k0 < kb; k0 += P * NW) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (k0 + p * NW >= kb) break;
            Step& s = st[p];
            FragOf<T> w[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) w[i].set(join(s.w[i][0], s.w[i][1]));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float up = s.sb * kScaleUp, up2 = s.sb2 * kScaleUp, f = s.sa[j] * up, f2 = s.sa[j] * up2;
                beyond = beyond || too_large(up) || too_large(f) || too_large(up2) || too_large(f2);
                FragOf<T> x;
                x.set(join(s.x[j][0], s.x[j][1]));
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const f32x4_t t = dot(w[i], x);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[i][j][r] = __builtin_fmaf(t[r], MODE == kGlu && i >= 2 ? f2 : f, acc[i][j][r]);
                }
            }
            if (k0 + (p + P) * NW < kb) load(k0 + (p + P) * NW, s);
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) s_part[wave][i][j][lane] = acc[i][j] * kScaleDown;
    if (__any(beyond))
        sum_any_scales<T, MODE, NI, NT>(a, bt, at, as, bs, (int64_t)hb * kb, a.N - 1 - n0, rows_m - 1, wave, NW,
                                        [&](int i, int j, const f32x4_t& v) { s_part[wave][i][j][lane] = v; });
    __syncthreads();
    if constexpr (MODE == kGlu) {
        static_assert(MODE != kGlu || NI == 4, "32 gate rows and their 32 up rows");
        float* h = static_cast<float*>(a.y);
        for (int it = wave; it < 2 * NT; it += NW) {
            const int i = it % 2, j = it / 2, at = n0 + i * 16 + 4 * lq, hc = n0 / 2 + i * 16 + 4 * lq;
            f32x4_t g = s_part[0][i][j][lane], u = s_part[0][(i + 2) % NI][j][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) {
                g += s_part[w][i][j][lane];
                u += s_part[w][(i + 2) % NI][j][lane];
            }
            f32x4_t o;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                o[r] = hc + r < a.hidden ? swiglu<__bf16>(g[r] + a.bias[at + r], u[r] + a.bias[at + 32 + r]) : 0.0f;
            const int m = j * 16 + l16;
            if (m < rows_m) *reinterpret_cast<f32x4_t*>(h + (m0 + m) * (a.N / 2) + hc) = o;
        }
        return;
    }
    T* y = static_cast<T*>(a.y);
    const bool whole = a.N % 4 == 0;
    for (int it = wave; it < NI * NT; it += NW) {
        const int i = it % NI, j = it / NI;
        f32x4_t v = s_part[0][i][j][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += s_part[w][i][j][lane];
        const int n = n0 + i * 16 + 4 * lq, m = j * 16 + l16;
        if (a.bias)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += n + r < a.N ? a.bias[n + r] : 0.0f;
        if (m < rows_m && n < a.N) put4(y + (m0 + m) * a.N, n, a.N, v, whole);
    }
}

template <typename T, int MODE, int NI, int NJ, int WN, int WM>
hipError_t tile(const Fp8GemmArgs& a, hipStream_t s) {
    const int64_t tm = (a.M + 16 * NJ * WM - 1) / (16 * NJ * WM), tn = (a.N + 16 * NI * WN - 1) / (16 * NI * WN);
    if (tm * tn >= ((int64_t)1 << 32) / (WN * WM * kWave) - kNumXcd) return hipErrorInvalidValue;
    launch_kernel(fp8_tile_kernel<T, MODE, NI, NJ, WN, WM>, dim3((unsigned)round_up(tm * tn, kNumXcd)),
                  dim3(WN * WM * kWave), 0, s, a, (int)tm, (int)tn);
    return hipGetLastError();
}
template <typename T, int MODE, int NI, int NT, int NW, int P>
hipError_t rows(const Fp8GemmArgs& a, hipStream_t s) {
    const int64_t tm = (a.M + 16 * NT - 1) / (16 * NT), tn = (a.N + 16 * NI - 1) / (16 * NI);
    if (tm > 65535) return hipErrorInvalidValue;
    launch_kernel(fp8_rows_kernel<T, MODE, NI, NT, NW, P>, dim3((unsigned)tn, (unsigned)tm), dim3(NW * kWave), 0, s, a);
    return hipGetLastError();
}

// Weight rows (16 NI) of a block of the kernel for few rows: as many as leave a block for each CU.
template <int NT>
int rows_ni(int64_t M, int N) {
    const int64_t tm = (M + 16 * NT - 1) / (16 * NT);
    return (N + 63) / 64 * tm >= 256 ? 4 : (N + 31) / 32 * tm >= 256 ? 2 : 1;
}
constexpr int rows_waves(int ni, int nt) { return ni == 4 && nt == 4 ? 4 : 8; }
template <typename T, int NT>
hipError_t few_rows(const Fp8GemmArgs& a, hipStream_t s) {
    switch (rows_ni<NT>(a.M, a.N)) {
        case 4: return rows<T, kStore, 4, NT, rows_waves(4, NT), 2>(a, s);
        case 2: return rows<T, kStore, 2, NT, 8, 2>(a, s);
    }
    return rows<T, kStore, 1, NT, 8, 2>(a, s);
}

// Up to 32 rows the kernel for few rows; more: the least estimate, in us, from rounds of 256 CUs and steps of 128
// columns. Measured in bf16 (few rows in tiles of 64; tiles of 128 x 128; of 256 x 256): 128 x 8,192 x 2,048 14.6, 18.1,
// 31.9; 512 x 8,192 x 2,048 51, 20.4, 33; 256 x 2,048 x 2,048 10.7, 17.6, 31; 40 x 2,048 x 8,192 22, 56, 106; 2,048 x 8,192
// x 2,048 190, 50, 40; 4,744 x 4,096 x 2,048 -, 58, 68; 4,744 x 2,048 x 8,192 -, 138, 113; 14,232 x 8,192 x 2,048 -, 326, 247.
// f32 results take twice the MFMA time and registers for widened fragments. Measured (few rows; tiles of 128 x 128; of
// 256 weight rows x 128, which were 24% slower to 2% faster and are not built): 128 x 8,192 x 2,048 16.8, 23.7, 32.7;
// 256 x 2,048 x 8,192 34, 78, 116; 1,024 x 1,536 x 4,096 48, 43, 63; 2,048 x 512 x 1,008 9.0, 14.5, 19.7; 4,744 x 2,048 x 8,192
// -, 188, 233; 14,232 x 8,192 x 2,048 -, 497, 488.
template <typename T>
hipError_t gemm(const Fp8GemmArgs& a, hipStream_t s) {
    if (a.M <= 16) return few_rows<T, 1>(a, s);
    if (a.M <= 32) return few_rows<T, 2>(a, s);
    const double kt = (a.K + kFp8Block - 1) / kFp8Block;
    auto rounds = [&](int bm, int bn) { return (double)(((a.M + bm - 1) / bm * ((a.N + bn - 1) / bn) + 255) / 256); };
    const int ni = rows_ni<4>(a.M, a.N);
    const double walk = std::ceil(kt / rows_waves(ni, 4)), r64 = rounds(64, 16 * ni), r128 = rounds(128, 128);
    if constexpr (sizeof(T) == 4) {
        const double few = 2 + r64 * (ni == 4 ? 3 + 2.6 * walk : ni == 2 ? 1.3 + 3.85 * walk : 3.4 * walk);
        const double t128 = 4 + kt * (r128 <= 1 ? 1.17 : 1.05 * r128);
        if (few <= t128 && a.M <= 65535 * 64) return few_rows<T, 4>(a, s);
        return tile<T, kStore, 4, 4, 2, 2>(a, s);
    } else {
        const double few = 5 + r64 * (2 + 2.2 * walk);
        const double t128 = 4 + kt * (r128 <= 1 ? 0.78 : 0.7 * r128), t256 = 4 + rounds(256, 256) * (3 + 1.65 * kt);
        if (few <= t128 && few <= t256 && a.M <= 65535 * 64) return few_rows<T, 4>(a, s);
        if (t128 <= t256) return tile<T, kStore, 4, 4, 2, 2>(a, s);
        return tile<T, kStore, 8, 4, 2, 4>(a, s);
    }
}

}  // namespace

hipError_t launch_fp8_gemm(DType dt, const Fp8GemmArgs& a, hipStream_t s) {
    // (a tile's bytes are addressed with 32 bits)
    if (a.M < 1 || a.N < 1 || a.K < 16 || a.K % 16 != 0 || a.K > kFp8MaxK || a.N > kFp8MaxN ||
        a.M > kFp8MaxRows)
        return hipErrorInvalidValue;
    switch (dt) {
        case DType::F32: return gemm<float>(a, s);
        case DType::BF16: return gemm<__bf16>(a, s);
        case DType::F16: return gemm<_Float16>(a, s);
    }
    return hipErrorInvalidValue;
}

bool fp8_glu_fused(int64_t M, int) { return M > kFp8GluRows; }

// Each rounding to 8 bits that falls the other way moves a hidden value by 1/16, so the hidden activations
// are made more exactly than the outputs: sums of 16-bit accuracy took the error of a feed-forward in
// f16 from 2.1e-4 to 22e-4 (515 rows, 96 x 2,093).  f32 sums cost a call of few rows nothing, which waits
// for its weights, and one of many a third (4,744 rows, 2,048 x 8,192: 312 -> 460 us): there bf16's, whose
// own rounding of the outputs is 17e-4, stay with the 8-bit instructions (17e-4 to 23e-4).
hipError_t launch_fp8_glu(DType dt, const Fp8GemmArgs& a, hipStream_t s) {
    if (a.M < 1 || a.N < 256 || a.N % 256 != 0 || a.K < 128 || a.K % 128 != 0 || a.K > kFp8MaxK || a.N > kFp8MaxN ||
        a.M > kFp8MaxRows || a.hidden < 1 || a.hidden > a.N / 2 || !a.bias)
        return hipErrorInvalidValue;
    if (!fp8_glu_fused(a.M, a.N)) {
        if (a.M <= 16) return rows<float, kGlu, 4, 1, 8, 2>(a, s);
        if (a.M <= 32) return rows<float, kGlu, 4, 2, 8, 2>(a, s);
        return rows<float, kGlu, 4, 4, 4, 2>(a, s);
    }
    if (dt != DType::BF16) return tile<float, kGlu, 8, 2, 2, 4>(a, s);
    // Tiles of 128 rows while they are one round of the CUs, else of 256 (us a feed-forward, 128 and 256 rows a tile: 512 rows
    // of 2,048 x 8,192, 256 tiles, 75 and 85; 4,744 of 512 x 512, 152 tiles, 28 and 34; 1,500 of 1,536 x 4,096, 384 tiles, 79
    // and 71; 9,000 of 2,048 x 512, 284 tiles, 87 and 77; 4,744 of 2,048 x 8,192 358 and 308).
    if ((a.M + 127) / 128 * (a.N / 256) <= 256) return tile<__bf16, kGlu, 8, 2, 2, 4>(a, s);
    return tile<__bf16, kGlu, 8, 4, 2, 4>(a, s);
}

}  // namespace nomas
