// The seam between two branches of a DiT block:
//
//   n   = y, or its RMS norm: y rsqrt(mean(y^2) + eps) post_w   (the branch's output)
//   out = alpha x + gate n
//   h   = out rsqrt(mean(out^2) + eps) norm_w (1 + scale) + shift
//
// Everything between the tensors is f32: one rounding to the model dtype per
// output, and h is made from out before that rounding.  Sums over a row are
// trees, not the serial chain of norm_modulate (seam.hip), whose bits are the
// reference's.
//
// HBM bound: x and y are read once, out and h written once (4 rows D elements).  A
// row stays in registers from its load to its stores, the parameters for
// all rows of a block's chunk.  18,720 rows of 2,560 f16: 76.9 us, 5.0 TB/s (a large copy reaches
// 5.1); 14,232 rows of 1,536 bf16 with both norms: 32 us (the last-level cache holds some of it).
#include "block_seam.hpp"

namespace nomas {

namespace {

// Blocks and threads of a call that fills the chip: enough waves for the loads in
// flight, rows enough per block for its parameters to be read from L2 seldom.  18,720
// rows of 2,560 f16 (383 MB): 1,024 blocks 81.9 us, 2,048 80.8, 4,096 76.9 (5.0 TB/s, what a
// large copy reaches); rows one or four at a time, or blocks of 512 threads: as long or longer.
constexpr int64_t kForwardBlocks = 4096;
constexpr int kForwardThreads = 256;

template <typename T, bool kPost, bool kNorm, int L, int C>
__global__ __launch_bounds__(kSeamThreads) void block_seam_kernel(BlockSeamArgs a, SeamPlan p) {
    constexpr int R = sizeof(T) == 4 || C > 1 ? 1 : 2;  // rows of a step
    __shared__ __align__(16) float s_part[sums_floats<L, R>()];
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
    const T* x = static_cast<const T*>(a.x);
    const T* y = static_cast<const T*>(a.y);
    T* out = static_cast<T*>(a.out);
    T* h = static_cast<T*>(a.h);
    const float inv_d = 1.0f / (float)D;

    // gate and post_w as one factor of y, norm_w and scale as one of out
    float gw[C][8], f[C][8], sh[C][8];
    auto params = [&](int64_t b) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float w[8];
            params8(a.gate, b * D + col[c], 1.0f, gw[c]);
            if constexpr (kPost) {
                params8(a.post_w, col[c], 1.0f, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) gw[c][i] *= w[i];
            }
            if constexpr (kNorm) {
                params8(a.scale, b * D + col[c], 0.0f, f[c]);
                params8(a.norm_w, col[c], 1.0f, w);
                params8(a.shift, b * D + col[c], 0.0f, sh[c]);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[c][i] = w[i] * (1.0f + f[c][i]);
            }
        }
    };
    int turn = 0;
    // rows at, at + stride, ... of those below `end`; all lanes run the same steps:
    // past the end the last row is computed again and not stored, nor anything
    // by a group that has nothing to do
    auto step = [&](int64_t at, int64_t stride, int64_t end, bool busy) {
        Raw8<T> rx[R][C], ry[R][C];
        int64_t row[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            row[r] = min(at + r * stride, end - 1);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                ry[r][c] = fetch8(y + row[r] * D, col[c]);
                rx[r][c] = fetch8(x + row[r] * D, col[c]);
            }
        }
        float v[R][C][8], s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                widen8(ry[r][c], v[r][c]);
                float q = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) q += v[r][c][i] * v[r][c][i];
                s[r] += live[c] ? q : 0.0f;
            }
        }
        if constexpr (kPost) row_sums<L>(s, s_part, turn++, W / kWave);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float n = kPost ? rsqrtf(s[r] * inv_d + a.eps) : 1.0f;
            s[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float u[8], q = 0.0f;
                widen8(rx[r][c], u);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[r][c][i] = a.alpha * u[i] + gw[c][i] * (v[r][c][i] * n);
                    q += v[r][c][i] * v[r][c][i];
                }
                s[r] += live[c] ? q : 0.0f;
                if (live[c] && busy && at + r * stride < end) put8(out + row[r] * D, col[c], v[r][c]);
            }
        }
        if constexpr (kNorm) {
            row_sums<L>(s, s_part, turn++, W / kWave);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float n = rsqrtf(s[r] * inv_d + a.eps);
#pragma unroll
                for (int c = 0; c < C; ++c) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[r][c][i] = v[r][c][i] * n * f[c][i] + sh[c][i];
                    if (live[c] && busy && at + r * stride < end) put8(h + row[r] * D, col[c], v[r][c]);
                }
            }
        }
    };
    if (p.whole) {
        const int64_t n = a.rows / a.seq;
        for (int64_t b0 = blockIdx.x * (int64_t)G; b0 < n; b0 += gridDim.x * (int64_t)G) {
            const int64_t b = min(b0 + g, n - 1);
            params(b);
            for (int64_t s = 0; s < a.seq; s += R) step(b * a.seq + s, 1, (b + 1) * a.seq, b0 + g < n);
        }
    } else {
        const int64_t b = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
        const int64_t first = b * a.seq + part * p.chunk, end = min(first + p.chunk, (b + 1) * a.seq);
        params(b);
        for (int64_t at = first; at < end; at += (int64_t)G * R) step(at + g, G, end, true);
    }
}

template <typename T>
hipError_t launch_seam_t(const BlockSeamArgs& a, hipStream_t s) {
    const SeamPlan p = seam_plan(a.rows, a.D, a.seq, kForwardBlocks, kForwardThreads);
    return with_seam_shape(p, [&](auto l, auto c) {
        constexpr int L = decltype(l)::value, C = decltype(c)::value;
        auto kern = a.post ? (a.h ? block_seam_kernel<T, true, true, L, C> : block_seam_kernel<T, true, false, L, C>)
                           : (a.h ? block_seam_kernel<T, false, true, L, C> : block_seam_kernel<T, false, false, L, C>);
        launch_kernel(kern, dim3((unsigned)p.blocks), dim3(p.row_threads * p.groups), 0, s, a, p);
        return hipGetLastError();
    });
}

}  // namespace

hipError_t launch_block_seam(DType dt, const BlockSeamArgs& a, hipStream_t s) {
    if (a.D < 8 || a.D % 8 != 0 || a.D > kMaxSeamDim || a.rows < 1 || a.rows > kMaxSeamRows || a.seq < 1 ||
        a.rows % a.seq != 0)
        return hipErrorInvalidValue;
    switch (dt) {
        case DType::F32: return launch_seam_t<float>(a, s);
        case DType::BF16: return launch_seam_t<__bf16>(a, s);
        case DType::F16: return launch_seam_t<_Float16>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace nomas
