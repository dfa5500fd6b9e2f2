// The gradients of the block seam (block_seam.hip).  Of the rows, with
// r = 1 / rms(out), ry = 1 / rms(y) (1 without the norm after the branch),
// f = norm_w (1 + scale), u = gate post_w:
//
//   d  = dout + r (dh f - out r c1),     c1 = mean(dh f out r)
//   dx = alpha d
//   dy = ry (u d - y ry c2),             c2 = mean(u d y ry)      (u d without the norm)
//
// and of the parameters, summed over the rows of a sequence,
//
//   P = sum dh, Q = sum dh out r, R = sum d y ry
//   dshift = P, dscale = norm_w Q, dgate = post_w R,
//   dnorm_w = sum over sequences of (1 + scale) Q, dpost_w = of gate R
//
// HBM bound: dout, dh, out and y are read once, dx and dy written once (6 rows D
// elements).  One pass does it all: c2's sum needs d, and d needs c1, but it is
// linear in d, so that sums of the inputs alone (out^2, y^2, dh f out, u y dout,
// u y dh f, u y out) give r, ry, c1 and c2 after one exchange per row.  P, Q and
// R grow in the registers of the threads that own the columns; each block
// leaves its sums in the workspace, and seam_sums_kernel adds them up in a
// fixed order: no atomics, the same bits every time.
//
// 14,232 rows of 1,536 bf16 (262 MB and 9 MB of sums): 60 us, 4.5 TB/s, and 5.6 for the sums; 5,998 rows of
// 1,000 f32: 32 us and 4.6.  Loading the next row ahead takes registers that are worth more
// as waves (114 us), a wave a row of three chunks a lane measured 58.5 and 37 us.  At 128 registers
// the bf16 form with both norms spills 6 of them (28 bytes of scratch a lane), narrow f32 rows 2.
// Rows past 8,192 columns hold four chunks a thread and spill 86 to 387 with both norms: 2,000 rows of 16,384
// take 195 us in bf16 and 306 in f32 (1.8 and 2.4 TB/s with the sums).
#include "block_seam.hpp"

namespace nomas {

namespace {

// Blocks and threads of a call that fills the chip: two blocks a CU, at 128 registers
// all of them at once where a block has six waves (768 or 1,536 columns, or narrow rows).  Each leaves 12 D
// bytes of sums, written and read again: 1,024 smaller blocks took as long, 768 blocks, of which a third run
// in a second round, 83 us where 512 took 60 (14,232 rows of 1,536 bf16).
// What the fixed number costs: rows of 2,048 columns have four waves a block, of 2,560 five, so that a CU is not
// full (14,232 rows: 89 us, 3.9 TB/s, and 109, 4.0); and a number of sequences that does not divide 512 passes it,
// since parts are rounded up (3 x 8,192 rows of 1,536 in 513 blocks 129 us, 3.5 TB/s; 24 x 592 in 528, 84 us, 3.1;
// 3 x 4,744 in 510, 60 us, 4.4).
constexpr int64_t kGradBlocks = 512;
constexpr int kGradThreads = 384;

// sums of a block's (or sequence's) columns: P, Q, R, each D floats
constexpr int kSums = 3;

// LDS: the parameters of a block's sequence, f and u [D] each, and later a group's
// sums of eight columns a thread.
__host__ __device__ inline uint32_t grad_lds(const SeamPlan& p, int D) {
    const uint32_t params = p.whole ? 0 : 2 * (uint32_t)D * 4, sums = (uint32_t)(p.row_threads * p.groups) * 8 * 4;
    return params > sums ? params : sums;
}

template <typename T, bool kPost, bool kNorm, bool kWhole, int L, int C>
__global__ __launch_bounds__(kSeamThreads) __attribute__((amdgpu_waves_per_eu(C == 1 && !kWhole ? 4 : 2)))
void seam_grad_kernel(BlockSeamBackwardArgs a, SeamPlan p, float* sums) {
    constexpr int N = (kNorm ? 2 : 0) + (kPost ? 2 : 0) + (kNorm && kPost ? 2 : 0);
    constexpr int NS = N ? N : 1;
    __shared__ __align__(16) float s_part[sums_floats<L, NS>()];
    extern __shared__ __align__(16) float s_dyn[];
    const int D = a.D;
    const int W = L ? L : p.row_threads, G = p.groups;
    // (the same for a wave where a row takes whole ones)
    const int g = L && L < 64 ? threadIdx.x / W : __builtin_amdgcn_readfirstlane(threadIdx.x / W);
    const int t = threadIdx.x - g * W;
    int col[C];
    bool live[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        live[c] = (t + c * W) * kSeamCols < D;
        col[c] = live[c] ? (t + c * W) * kSeamCols : 0;
    }
    const T* dout = static_cast<const T*>(a.dout);
    const T* dh = static_cast<const T*>(a.dh);
    const T* out = static_cast<const T*>(a.out);
    const T* y = static_cast<const T*>(a.y);
    T* dx = static_cast<T*>(a.dx);
    T* dy = static_cast<T*>(a.dy);
    const float inv_d = 1.0f / (float)D;

    // f = norm_w (1 + scale) and u = gate post_w for eight columns of sequence b
    auto factors = [&](int64_t b, int at, float* f, float* u) {
        float w[8];
        params8(a.gate, b * D + at, 1.0f, u);
        if constexpr (kPost) {
            params8(a.post_w, at, 1.0f, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] *= w[i];
        }
        if constexpr (kNorm) {
            params8(a.scale, b * D + at, 0.0f, f);
            params8(a.norm_w, at, 1.0f, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = w[i] * (1.0f + f[i]);
        }
    };
    float own[2][kWhole ? C : 1][8];  // kWhole: this group's f and u (else they are in LDS)
    auto get_f = [&](int c, float* f) {
        if constexpr (kWhole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = own[0][c][i];
        } else {
            load_f32s<8>(s_dyn + col[c], f);
        }
    };
    auto get_u = [&](int c, float* u) {
        if constexpr (kWhole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = own[1][c][i];
        } else {
            load_f32s<8>(s_dyn + D + col[c], u);
        }
    };
    float acc[kSums][C][8];
    auto clear = [&](float (&v)[C][8]) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0.0f;
    };
    clear(acc[0]);
    clear(acc[1]);
    clear(acc[2]);
    int turn = 0;
    // One row of each group; `on`: it is a row of this group (all lanes run the same
    // steps, those without a row compute one that nothing is kept of).
    auto step = [&](int64_t row, bool on) {
        const int64_t o = row * D;
        Raw8<T> rd[C], rh[C], ro[C], ry[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if constexpr (kNorm) {
                rh[c] = fetch8(dh + o, col[c]);
                ro[c] = fetch8(out + o, col[c]);
            }
            rd[c] = {};
            if (dout) rd[c] = fetch8(dout + o, col[c]);
            ry[c] = {};
            if (kPost || y) ry[c] = fetch8(y + o, col[c]);
        }
        float m[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) m[i] = 0.0f;
        if constexpr (N > 0) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float vo[8], vh[8], vy[8], vd[8], f[8], u[8], q[N];
#pragma unroll
                for (int i = 0; i < N; ++i) q[i] = 0.0f;
                if constexpr (kNorm) {
                    widen8(rh[c], vh);
                    widen8(ro[c], vo);
                    get_f(c, f);
                }
                if constexpr (kPost) {
                    widen8(ry[c], vy);
                    widen8(rd[c], vd);
                    get_u(c, u);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (kNorm) {
                        vh[i] *= f[i];
                        q[0] += vo[i] * vo[i];
                        q[1] += vh[i] * vo[i];
                    }
                    if constexpr (kPost) {
                        constexpr int k = kNorm ? 2 : 0;
                        q[k] += vy[i] * vy[i];
                        const float uy = u[i] * vy[i];
                        q[k + 1] += uy * vd[i];
                        if constexpr (kNorm) {
                            q[k + 2] += uy * vh[i];
                            q[k + 3] += uy * vo[i];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < N; ++i) m[i] += live[c] ? q[i] : 0.0f;
            }
            row_sums<L>(m, s_part, turn++, W / kWave);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                renew(rd[c]);
                renew(ry[c]);
                if constexpr (kNorm) {
                    renew(rh[c]);
                    renew(ro[c]);
                }
            }
        }
        if (!on) return;
        float r = 0.0f, k1 = 0.0f, iy = 1.0f, k2 = 0.0f;
        if constexpr (kNorm) {
            r = rsqrtf(m[0] * inv_d + a.eps);
            k1 = r * (r * (r * (m[1] * inv_d)));  // of out in d (r^3 by itself leaves f32's range at rms 1e13)
        }
        if constexpr (kPost) {
            constexpr int k = kNorm ? 2 : 0;
            iy = rsqrtf(m[k] * inv_d + a.eps);
            float dot = m[k + 1];
            if constexpr (kNorm) dot += r * m[k + 2] - k1 * m[k + 3];
            k2 = iy * (iy * (dot * inv_d));  // of y in dy / iy
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!live[c]) continue;
            float d[8], v[8];
            widen8(rd[c], d);
            if constexpr (kNorm) {
                float vo[8], vh[8], f[8];
                widen8(rh[c], vh);
                widen8(ro[c], vo);
                get_f(c, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    acc[0][c][i] += vh[i];
                    vh[i] *= r;
                    acc[1][c][i] += vh[i] * vo[i];
                    d[i] += vh[i] * f[i] - k1 * vo[i];
                }
            }
            if (kPost || y) {
                float vy[8], w[8], u[8];
                widen8(ry[c], vy);
                get_u(c, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    acc[2][c][i] += (iy * d[i]) * vy[i];
                    w[i] = kPost ? iy * (d[i] * u[i] - k2 * vy[i]) : d[i] * u[i];
                }
                if (dy) put8(dy + o, col[c], w);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = a.alpha * d[i];
            if (dx) put8(dx + o, col[c], v);
        }
    };
    // The groups' values of the columns added up, in the first group's lanes: by
    // eights, every group's in LDS, in the groups' order.
    auto over_groups = [&](float (&v)[C][8]) {
        if (G == 1) return;
        const int n = W * G;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) s_dyn[i * n + threadIdx.x] = v[c][i];
            __syncthreads();
            if (g == 0)
                for (int q = 1; q < G; ++q)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[c][i] += s_dyn[i * n + q * W + t];
        }
    };
    if constexpr (kWhole) {
        const int64_t n = a.rows / a.seq;
        float gain[2][C][8];  // of norm_w and post_w
        clear(gain[0]);
        clear(gain[1]);
        for (int64_t b0 = blockIdx.x * (int64_t)G; b0 < n; b0 += gridDim.x * (int64_t)G) {
            const bool busy = b0 + g < n;
            const int64_t b = min(b0 + g, n - 1);
#pragma unroll
            for (int c = 0; c < C; ++c) factors(b, col[c], own[0][c], own[1][c]);
            for (int64_t s = 0; s < a.seq; ++s) step(b * a.seq + s, busy);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (!busy || !live[c]) continue;
                const int64_t o = b * D + col[c];
                float w[8], v[8];
                params8(a.norm_w, col[c], 1.0f, w);
                if (a.dshift) put8(a.dshift + o, acc[0][c]);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = w[i] * acc[1][c][i];
                if (a.dscale) put8(a.dscale + o, v);
                params8(kPost ? a.post_w : nullptr, col[c], 1.0f, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = w[i] * acc[2][c][i];
                if (a.dgate) put8(a.dgate + o, v);
                params8(a.scale, o, 0.0f, w);
                params8(a.gate, o, 1.0f, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    gain[0][c][i] += (1.0f + w[i]) * acc[1][c][i];
                    gain[1][c][i] += v[i] * acc[2][c][i];
                }
            }
            clear(acc[0]);
            clear(acc[1]);
            clear(acc[2]);
        }
        over_groups(gain[0]);
        over_groups(gain[1]);
        if (g == 0) {
            float* o = sums + blockIdx.x * 2 * (int64_t)D;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (live[c]) {
                    put8(o + col[c], gain[0][c]);
                    put8(o + D + col[c], gain[1][c]);
                }
        }
    } else {
        const int64_t b = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
        const int64_t first = b * a.seq + part * p.chunk, end = min(first + p.chunk, (b + 1) * a.seq);
        for (int at = threadIdx.x * kSeamCols; at < D; at += blockDim.x * kSeamCols) {
            float f[8], u[8];
            factors(b, at, f, u);
            if constexpr (kNorm) put8(s_dyn + at, f);
            put8(s_dyn + D + at, u);
        }
        __syncthreads();
        for (int64_t at = first; at < end; at += G) step(min(at + g, end - 1), at + g < end);
        over_groups(acc[0]);
        over_groups(acc[1]);
        over_groups(acc[2]);
        if (g == 0) {
            float* o = sums + blockIdx.x * kSums * (int64_t)D;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (live[c])
#pragma unroll
                    for (int k = 0; k < kSums; ++k) put8(o + k * (int64_t)D + col[c], acc[k][c]);
        }
    }
}

// ---- the blocks' sums added up ----
//
// A block takes 32 columns (8 threads of four each) of one of the sums, blockIdx.z; the
// rows of sums are dealt out to 64 slices, eight a wave.  32 columns are a line of 128 bytes:
// with 16, and 128 slices in twice the blocks, the 512 rows of 1,536 take 7.5 us instead of 5.5.

constexpr int kSumSlices = 64, kSumQuads = 8, kSumThreads = kSumSlices * kSumQuads;
constexpr int kSumWaves = kSumThreads / kWave, kSumWaveSlices = kSumSlices / kSumWaves;
// Sequences whose sums one block adds, so that it can finish the gains too.
constexpr int kSumSeqs = 4;

__device__ __forceinline__ void add4(float4& v, const float4& o) {
    v.x += o.x;
    v.y += o.y;
    v.z += o.z;
    v.w += o.w;
}

// v[i], i < seqs: the sum of rows slice, slice + slices, ... of the m rows of sequence i
// (`pitch` floats apart), added over the slices that the wave holds.  The loads of a
// flight, of all sequences, are unconditional, clamped to the last row: they wait once.
template <int N>
__device__ __forceinline__ void sum_rows(const float* p, int64_t m, int64_t pitch, int seqs, int slice, int slices,
                                         float4 (&v)[N]) {
    constexpr int kFlight = 4;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int64_t r = slice; r < m; r += kFlight * slices) {
        float4 o[N][kFlight];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < seqs)
#pragma unroll
                for (int j = 0; j < kFlight; ++j)
                    o[i][j] = *reinterpret_cast<const float4*>(p + (i * m + min(r + j * slices, m - 1)) * pitch);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < kFlight; ++j)
                if (i < seqs && r + j * slices < m) add4(v[i], o[i][j]);
    }
    // lanes with the same columns are 8, 16 and 32 apart
    auto over_slices = [](float x) {
        x = dpp_add<0x128>(x);  // row_ror: 8
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
        const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return __uint_as_float(t[0]) + __uint_as_float(t[1]);
    };
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < seqs) v[i] = make_float4(over_slices(v[i].x), over_slices(v[i].y), over_slices(v[i].z), over_slices(v[i].w));
}

// x times four of w (1 where there is none), or of 1 + w (w 0 where there is none)
__device__ __forceinline__ float4 times(const float4& x, const float* w, bool plus_one) {
    if (!w) return x;
    float4 g = *reinterpret_cast<const float4*>(w);
    const float c = plus_one ? 1.0f : 0.0f;
    return make_float4((c + g.x) * x.x, (c + g.y) * x.y, (c + g.z) * x.z, (c + g.w) * x.w);
}
__device__ __forceinline__ void put4(float* to, const float4& x) { *reinterpret_cast<float4*>(to) = x; }

// From x, sum k (P, Q, R) of four columns of sequence b: that parameter's gradient; what
// it adds to the gradient of norm_w (Q) or post_w (R) is returned.
__device__ __forceinline__ float4 finish_sequence(const BlockSeamBackwardArgs& a, int k, int64_t b, int col, const float4& x) {
    const int64_t o = b * a.D + col;
    if (k == 0) {
        if (a.dshift) put4(a.dshift + o, x);
        return x;
    }
    if (k == 1) {
        if (a.dscale) put4(a.dscale + o, times(x, a.norm_w ? a.norm_w + col : nullptr, false));
        return times(x, a.scale ? a.scale + o : nullptr, true);
    }
    if (a.dgate) put4(a.dgate + o, times(x, a.post && a.post_w ? a.post_w + col : nullptr, false));
    return times(x, a.gate ? a.gate + o : nullptr, false);
}

// n <= kSumSeqs sequences of `parts` rows [3][D]: all gradients of parameters.
__global__ __launch_bounds__(kSumThreads) void seam_sums_kernel(BlockSeamBackwardArgs a, const float* sums, int n,
                                                                int64_t parts) {
    __shared__ float4 s_v[kSumSeqs][kSumWaves][kSumQuads];
    const int q = threadIdx.x % kSumQuads, slice = threadIdx.x / kSumQuads, wave = threadIdx.x / kWave;
    const int col = (blockIdx.x * kSumQuads + q) * 4, k = blockIdx.z;
    const bool live = col < a.D;
    float4 v[kSumSeqs];
    sum_rows(sums + (int64_t)k * a.D + (live ? col : 0), parts, kSums * (int64_t)a.D, n, slice, kSumSlices, v);
#pragma unroll
    for (int i = 0; i < kSumSeqs; ++i)
        if ((threadIdx.x & 63) < kSumQuads) s_v[i][wave][q] = v[i];
    __syncthreads();
    // slice i's threads finish sequence i
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const bool mine = slice < n && live;
    if (mine) {
        for (int w = 0; w < kSumWaves; ++w) add4(x, s_v[slice][w][q]);
        x = finish_sequence(a, k, slice, col, x);
    }
    float* to = k == 0 ? nullptr : k == 1 ? a.dnorm_w : a.dpost_w;
    if (!to) return;
    __syncthreads();
    if (mine) s_v[slice][0][q] = x;
    __syncthreads();
    if (slice || !live) return;
    for (int i = 1; i < n; ++i) add4(x, s_v[i][0][q]);
    put4(to + col, x);
}

// More sequences, a wave each: their gradients, and the shares of the gains [n][2][D].
// (A block of 64 slices for each would stand idle where a sequence has few rows of sums:
// the backward pass of 64 x 16 rows of 1,536 takes 26 us, and took 45 so.)
__global__ __launch_bounds__(kSumThreads) void seam_sequence_sums_kernel(BlockSeamBackwardArgs a, const float* sums,
                                                                         int64_t n, int64_t parts, float* gains) {
    const int q = threadIdx.x % kSumQuads, slice = threadIdx.x % kWave / kSumQuads;
    const int col = (blockIdx.x * kSumQuads + q) * 4, k = blockIdx.z;
    const int64_t b = blockIdx.y * (int64_t)kSumWaves + threadIdx.x / kWave;
    if (b >= n) return;
    const bool live = col < a.D;
    float4 v[1];
    sum_rows(sums + (b * parts * kSums + k) * a.D + (live ? col : 0), parts, kSums * (int64_t)a.D, 1, slice,
             kSumWaveSlices, v);
    if (slice || !live) return;
    const float4 x = finish_sequence(a, k, b, col, v[0]);
    if (k) put4(gains + (b * 2 + k - 1) * a.D + col, x);
}

// Shares [n][2][D] of the gains, of sequences or of blocks: dnorm_w and dpost_w.
__global__ __launch_bounds__(kSumThreads) void seam_gain_sums_kernel(BlockSeamBackwardArgs a, const float* gains, int64_t n) {
    __shared__ float4 s_v[kSumWaves][kSumQuads];
    float* to = blockIdx.z ? a.dpost_w : a.dnorm_w;
    if (!to) return;
    const int q = threadIdx.x % kSumQuads, slice = threadIdx.x / kSumQuads;
    const int col = (blockIdx.x * kSumQuads + q) * 4;
    const bool live = col < a.D;
    float4 v[1];
    sum_rows(gains + (int64_t)blockIdx.z * a.D + (live ? col : 0), n, 2 * (int64_t)a.D, 1, slice, kSumSlices, v);
    if ((threadIdx.x & 63) < kSumQuads) s_v[threadIdx.x / kWave][q] = v[0];
    __syncthreads();
    if (slice || !live) return;
    for (int w = 1; w < kSumWaves; ++w) add4(v[0], s_v[w][q]);
    put4(to + col, v[0]);
}

__global__ __launch_bounds__(256) void zero_gains_kernel(float* p, float* q, int D) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= D) return;
    if (p) p[c] = 0.0f;
    if (q) q[c] = 0.0f;
}

SeamPlan grad_plan(int64_t rows, int64_t D, int64_t seq) {
    return seam_plan(rows, D, seq, kGradBlocks, kGradThreads);
}

template <typename T, bool kWhole, int L, int C>
hipError_t launch_grad_shape(const BlockSeamBackwardArgs& a, const SeamPlan& p, float* sums, hipStream_t s) {
    const bool norm = a.dh != nullptr, post = a.post && a.y;
    auto kern = post ? (norm ? seam_grad_kernel<T, true, true, kWhole, L, C> : seam_grad_kernel<T, true, false, kWhole, L, C>)
                     : (norm ? seam_grad_kernel<T, false, true, kWhole, L, C> : seam_grad_kernel<T, false, false, kWhole, L, C>);
    const uint32_t lds = grad_lds(p, a.D);
    if (lds > 48 * 1024) {
        // (the widest row's: calls of several threads set the same value)
        const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 2 * kMaxSeamDim * 4);
        if (e != hipSuccess) return e;
    }
    launch_kernel(kern, dim3((unsigned)p.blocks), dim3(p.row_threads * p.groups), lds, s, a, p, sums);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_grad_t(const BlockSeamBackwardArgs& a, hipStream_t s) {
    const SeamPlan p = grad_plan(a.rows, a.D, a.seq);
    float* sums = static_cast<float*>(a.workspace);
    const hipError_t e =
        p.whole ? with_seam_shape(p, [&](auto l, auto c) {
            return launch_grad_shape<T, true, decltype(l)::value, decltype(c)::value>(a, p, sums, s);
        })
                : with_seam_shape(p, [&](auto l, auto c) {
                      return launch_grad_shape<T, false, decltype(l)::value, decltype(c)::value>(a, p, sums, s);
                  });
    if (e != hipSuccess || !(a.dgate || a.dshift || a.dscale || a.dnorm_w || a.dpost_w)) return e;
    const int64_t n = a.rows / a.seq;
    const unsigned cols = (unsigned)((a.D + 4 * kSumQuads - 1) / (4 * kSumQuads));
    const bool want_gains = a.dnorm_w || a.dpost_w;
    auto gain_sums = [&](const float* gains, int64_t rows) {
        if (want_gains)
            launch_kernel(seam_gain_sums_kernel, dim3(cols, 1, 2), dim3(kSumThreads), 0, s, a, gains, rows);
    };
    if (p.whole) {  // each block's shares of the gains
        gain_sums(sums, p.blocks);
    } else if (n <= kSumSeqs) {
        launch_kernel(seam_sums_kernel, dim3(cols, 1, kSums), dim3(kSumThreads), 0, s, a, (const float*)sums, (int)n,
                      p.parts);
    } else {
        float* gains = sums + p.blocks * kSums * a.D;
        launch_kernel(seam_sequence_sums_kernel, dim3(cols, (unsigned)((n + kSumWaves - 1) / kSumWaves), kSums),
                      dim3(kSumThreads), 0, s, a, (const float*)sums, n, p.parts, gains);
        gain_sums(gains, n);
    }
    return hipGetLastError();
}

}  // namespace

int64_t block_seam_workspace(int64_t rows, int64_t D, int64_t seq) {
    const SeamPlan p = grad_plan(rows, D, seq);
    const int64_t floats = p.whole ? p.blocks * 2 * D : (p.blocks * kSums + rows / seq * 2) * D;
    return floats * (int64_t)sizeof(float);
}

hipError_t launch_block_seam_backward(DType dt, const BlockSeamBackwardArgs& a, hipStream_t s) {
    if (a.D < 8 || a.D % 8 != 0 || a.D > kMaxSeamDim || a.rows < 0 || a.rows > kMaxSeamRows || a.seq < 1 ||
        a.rows % a.seq != 0)
        return hipErrorInvalidValue;
    if (a.rows == 0) {
        launch_kernel(zero_gains_kernel, dim3((a.D + 255) / 256), dim3(256), 0, s, a.dnorm_w, a.dpost_w, a.D);
        return hipGetLastError();
    }
    switch (dt) {
        case DType::F32: return launch_grad_t<float>(a, s);
        case DType::BF16: return launch_grad_t<__bf16>(a, s);
        case DType::F16: return launch_grad_t<_Float16>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace nomas
