// The seam between two branches of a DiT block, and its gradients:
//
//   n   = y, or its RMS norm: y rsqrt(mean(y^2) + eps) post_w   (the branch's output)
//   out = alpha x + gate n
//   h   = out rsqrt(mean(out^2) + eps) norm_w (1 + scale) + shift
//
// Everything between the tensors is f32: one rounding to the model dtype per
// output, and h is made from out before that rounding.  Sums over a row are
// trees, not the serial chain of norm_modulate (seam.hip), whose bits are the
// reference's.
#include <algorithm>

#include "kernels.hpp"
#include "seam.hpp"

namespace nomas {

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 8;  // columns that a thread takes at a time (D % 8 == 0)

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* o) {
    load16(p, o);
    if constexpr (sizeof(T) == 4) load16(p + 4, o + 4);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
    store16(p, v);
    if constexpr (sizeof(T) == 4) store16(p + 4, v + 4);
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

// The sums of N values over the block, in every thread.
template <int N>
__device__ void block_sums(float* v) {
    __shared__ float s_part[kThreads / kWave][N];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; ++i)
        for (int o = 32; o; o >>= 1) v[i] += __shfl_xor(v[i], o);
    __syncthreads();
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) s_part[wave][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0f;
        for (int w = 0; w < kThreads / kWave; ++w) v[i] += s_part[w][i];
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void block_seam_kernel(BlockSeamArgs a) {
    extern __shared__ float s_out[];  // the row of out, f32
    const int64_t row = blockIdx.x, p0 = row / a.seq * a.D;
    const T* x = static_cast<const T*>(a.x) + row * a.D;
    const T* y = static_cast<const T*>(a.y) + row * a.D;
    T* out = static_cast<T*>(a.out) + row * a.D;
    float ry = 1.0f;
    if (a.post) {
        float ss = 0.0f;
        for (int c = threadIdx.x * kCols; c < a.D; c += kThreads * kCols) {
            float v[8];
            load8(y + c, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += v[i] * v[i];
        }
        block_sums<1>(&ss);
        ry = rsqrtf(ss / a.D + a.eps);
    }
    float so = 0.0f;
    for (int c = threadIdx.x * kCols; c < a.D; c += kThreads * kCols) {
        float v[8], u[8], g[8], w[8];
        load8(x + c, v);
        load8(y + c, u);
        params8(a.gate, p0 + c, 1.0f, g);
        params8(a.post ? a.post_w : nullptr, c, 1.0f, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = a.alpha * v[i] + g[i] * (u[i] * ry * w[i]);
            so += v[i] * v[i];
            s_out[c + i] = v[i];
        }
        store8(out + c, v);
    }
    if (!a.h) return;
    block_sums<1>(&so);
    const float r = rsqrtf(so / a.D + a.eps);
    for (int c = threadIdx.x * kCols; c < a.D; c += kThreads * kCols) {
        float v[8], w[8], sc[8], sh[8];
        params8(a.norm_w, c, 1.0f, w);
        params8(a.scale, p0 + c, 0.0f, sc);
        params8(a.shift, p0 + c, 0.0f, sh);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = s_out[c + i] * r * w[i] * (1.0f + sc[i]) + sh[i];
        store8(static_cast<T*>(a.h) + row * a.D + c, v);
    }
}

// What a row's gradients need of the whole row.
struct RowStats {
    float r, c1;   // 1 / rms of out, mean(g out r)
    float ry, c2;  // of y, mean(gy y ry)
};

// dO and the branch's normalised output y ry for 8 columns of a row.
template <typename T>
__device__ __forceinline__ void grad8(const BlockSeamBackwardArgs& a, int64_t row, int c, const RowStats& st,
                                      float* d, float* yn, float* dh, float* unit) {
    const int64_t p = row / a.seq * a.D + c, at = row * a.D + c;
    float g[8], sc[8];
    params8(nullptr, 0, 0.0f, d);
    if (a.dout) load8(static_cast<const T*>(a.dout) + at, d);
    params8(nullptr, 0, 0.0f, dh);
    params8(nullptr, 0, 0.0f, unit);
    if (a.dh) {
        load8(static_cast<const T*>(a.dh) + at, dh);
        load8(static_cast<const T*>(a.out) + at, unit);
        params8(a.norm_w, c, 1.0f, g);
        params8(a.scale, p, 0.0f, sc);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            unit[i] *= st.r;
            d[i] += st.r * (dh[i] * (1.0f + sc[i]) * g[i] - unit[i] * st.c1);
        }
    }
    params8(nullptr, 0, 0.0f, yn);
    if (a.y) {
        load8(static_cast<const T*>(a.y) + at, yn);
#pragma unroll
        for (int i = 0; i < 8; ++i) yn[i] *= st.ry;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void seam_stats_kernel(BlockSeamBackwardArgs a, RowStats* stats) {
    const int64_t row = blockIdx.x;
    RowStats st = {1.0f, 0.0f, 1.0f, 0.0f};
    float v[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x * kCols; c < a.D; c += kThreads * kCols) {
        float d[8], yn[8], dh[8], unit[8];
        grad8<T>(a, row, c, st, d, yn, dh, unit);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[0] += unit[i] * unit[i];
            v[1] += yn[i] * yn[i];
        }
    }
    block_sums<2>(v);
    st.r = rsqrtf(v[0] / a.D + a.eps);
    if (a.post) st.ry = rsqrtf(v[1] / a.D + a.eps);
    float c1 = 0.0f;
    for (int c = threadIdx.x * kCols; c < a.D; c += kThreads * kCols) {
        float d[8], yn[8], dh[8], unit[8], w[8], sc[8];
        grad8<T>(a, row, c, st, d, yn, dh, unit);
        params8(a.norm_w, c, 1.0f, w);
        params8(a.scale, row / a.seq * a.D + c, 0.0f, sc);
#pragma unroll
        for (int i = 0; i < 8; ++i) c1 += dh[i] * (1.0f + sc[i]) * w[i] * unit[i];
    }
    block_sums<1>(&c1);
    st.c1 = c1 / a.D;
    if (a.post) {
        float c2 = 0.0f;
        for (int c = threadIdx.x * kCols; c < a.D; c += kThreads * kCols) {
            float d[8], yn[8], dh[8], unit[8], w[8], g[8];
            grad8<T>(a, row, c, st, d, yn, dh, unit);
            params8(a.post_w, c, 1.0f, w);
            params8(a.gate, row / a.seq * a.D + c, 1.0f, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) c2 += d[i] * g[i] * w[i] * yn[i];
        }
        block_sums<1>(&c2);
        st.c2 = c2 / a.D;
    }
    if (threadIdx.x == 0) stats[row] = st;
}

// Column sums of a sequence: shift's, and (before the gains) scale's and gate's.
template <typename T>
__global__ __launch_bounds__(kThreads) void seam_columns_kernel(BlockSeamBackwardArgs a, const RowStats* stats,
                                                                float* sums) {
    const int c = (blockIdx.x * kThreads + threadIdx.x) * kCols;
    const int64_t b = blockIdx.y, n = a.rows / a.seq;
    if (c >= a.D) return;
    float p[8] = {}, q[8] = {}, r[8] = {};
    for (int64_t row = b * a.seq; row < (b + 1) * a.seq; ++row) {
        float d[8], yn[8], dh[8], unit[8];
        grad8<T>(a, row, c, stats[row], d, yn, dh, unit);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] += dh[i];
            q[i] += dh[i] * unit[i];
            r[i] += d[i] * yn[i];
        }
    }
    float w[8], pw[8];
    params8(a.norm_w, c, 1.0f, w);
    params8(a.post ? a.post_w : nullptr, c, 1.0f, pw);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t at = b * a.D + c + i;
        if (a.dshift) a.dshift[at] = p[i];
        if (a.dscale) a.dscale[at] = q[i] * w[i];
        if (a.dgate) a.dgate[at] = r[i] * pw[i];
        sums[at] = q[i];
        sums[n * a.D + at] = r[i];
    }
}

__global__ __launch_bounds__(kThreads) void seam_gains_kernel(BlockSeamBackwardArgs a, const float* sums) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.D) return;
    const int64_t n = a.rows / a.seq;
    float dn = 0.0f, dp = 0.0f;
    for (int64_t b = 0; b < n; ++b) {
        dn += sums[b * a.D + c] * (1.0f + (a.scale ? a.scale[b * a.D + c] : 0.0f));
        dp += sums[(n + b) * a.D + c] * (a.gate ? a.gate[b * a.D + c] : 1.0f);
    }
    if (a.dnorm_w) a.dnorm_w[c] = dn;
    if (a.dpost_w) a.dpost_w[c] = dp;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void seam_rows_kernel(BlockSeamBackwardArgs a, const RowStats* stats) {
    const int64_t row = blockIdx.x;
    const RowStats st = stats[row];
    for (int c = threadIdx.x * kCols; c < a.D; c += kThreads * kCols) {
        float d[8], yn[8], dh[8], unit[8], g[8], w[8];
        grad8<T>(a, row, c, st, d, yn, dh, unit);
        params8(a.gate, row / a.seq * a.D + c, 1.0f, g);
        params8(a.post ? a.post_w : nullptr, c, 1.0f, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            g[i] *= d[i];
            if (a.post) g[i] = st.ry * (g[i] * w[i] - yn[i] * st.c2);
            d[i] *= a.alpha;
        }
        if (a.dx) store8(static_cast<T*>(a.dx) + row * a.D + c, d);
        if (a.dy) store8(static_cast<T*>(a.dy) + row * a.D + c, g);
    }
}

template <typename T>
hipError_t launch_seam_t(const BlockSeamArgs& a, hipStream_t s) {
    const int lds = a.D * 4;
    const hipError_t e = hipFuncSetAttribute((const void*)block_seam_kernel<T>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    launch_kernel(block_seam_kernel<T>, dim3((unsigned)a.rows), dim3(kThreads), lds, s, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_backward_t(const BlockSeamBackwardArgs& a, hipStream_t s) {
    RowStats* stats = static_cast<RowStats*>(a.workspace);
    float* sums = reinterpret_cast<float*>(stats + a.rows);
    const unsigned n = (unsigned)(a.rows / a.seq), cols = (a.D / kCols + kThreads - 1) / kThreads;
    if (a.rows == 0) {  // the gains' gradients are zero
        launch_kernel(seam_gains_kernel, dim3((a.D + kThreads - 1) / kThreads), dim3(kThreads), 0, s, a,
                      (const float*)nullptr);
        return hipGetLastError();
    }
    launch_kernel(seam_stats_kernel<T>, dim3((unsigned)a.rows), dim3(kThreads), 0, s, a, stats);
    launch_kernel(seam_columns_kernel<T>, dim3(cols, n), dim3(kThreads), 0, s, a, (const RowStats*)stats, sums);
    launch_kernel(seam_gains_kernel, dim3((a.D + kThreads - 1) / kThreads), dim3(kThreads), 0, s, a,
                  (const float*)sums);
    launch_kernel(seam_rows_kernel<T>, dim3((unsigned)a.rows), dim3(kThreads), 0, s, a, (const RowStats*)stats);
    return hipGetLastError();
}

}  // namespace

int64_t block_seam_workspace(int64_t rows, int64_t D, int64_t seq) {
    return rows * (int64_t)sizeof(RowStats) + 2 * (rows / seq) * D * (int64_t)sizeof(float);
}

hipError_t launch_block_seam(DType dt, const BlockSeamArgs& a, hipStream_t s) {
    if (a.D < 8 || a.D % 8 != 0 || a.D > kMaxSeamDim || a.rows < 1 || a.rows > kMaxSeamRows || a.seq < 1)
        return hipErrorInvalidValue;
    switch (dt) {
        case DType::F32: return launch_seam_t<float>(a, s);
        case DType::BF16: return launch_seam_t<__bf16>(a, s);
        case DType::F16: return launch_seam_t<_Float16>(a, s);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_block_seam_backward(DType dt, const BlockSeamBackwardArgs& a, hipStream_t s) {
    if (a.D < 8 || a.D % 8 != 0 || a.D > kMaxSeamDim || a.rows < 0 || a.rows > kMaxSeamRows || a.seq < 1 ||
        a.rows % a.seq != 0)
        return hipErrorInvalidValue;
    switch (dt) {
        case DType::F32: return launch_backward_t<float>(a, s);
        case DType::BF16: return launch_backward_t<__bf16>(a, s);
        case DType::F16: return launch_backward_t<_Float16>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace nomas
