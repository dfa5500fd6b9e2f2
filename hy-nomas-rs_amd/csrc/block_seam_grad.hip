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
#include "block_seam.hpp"

namespace nomas {

namespace {

// Blocks of a call that fills the chip.  Each leaves 12 D bytes of sums, written and
// read again.
#ifndef V_BLOCKS
#define V_BLOCKS 768
#endif
#ifndef V_PRE
#define V_PRE 1
#endif
#ifndef V_R
#define V_R 2
#endif
#ifndef V_GT
#define V_GT 512
#endif
constexpr int64_t kGradBlocks = V_BLOCKS;
constexpr int kGradThreads = V_GT;

// sums of a block's (or sequence's) columns: P, Q, R, each D floats
constexpr int kSums = 3;

template <typename T, bool kPost, bool kNorm, bool kWhole, int L, int C>
__global__ __launch_bounds__(kSeamThreads)
#ifdef V_WPE
__attribute__((amdgpu_waves_per_eu(C == 1 ? V_WPE : 2)))
#endif
void seam_grad_kernel(BlockSeamBackwardArgs a, SeamPlan p,
                                                                                float* sums) {
    constexpr int R = sizeof(T) == 4 || C > 1 ? 1 : V_R;     // rows of a step
    constexpr int N = (kNorm ? 2 : 0) + (kPost ? 2 : 0) + (kNorm && kPost ? 2 : 0);
    constexpr int NS = N ? N * R : 1;
    __shared__ __align__(16) float s_part[sums_floats<L, NS>()];
    __shared__ float s_v[kSeamThreads * 8];  // over_groups()
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

    float f[C][8], u[C][8];
    auto params = [&](int64_t b) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float w[8];
            params8(a.gate, b * D + col[c], 1.0f, u[c]);
            if constexpr (kPost) {
                params8(a.post_w, col[c], 1.0f, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[c][i] *= w[i];
            }
            if constexpr (kNorm) {
                params8(a.scale, b * D + col[c], 0.0f, f[c]);
                params8(a.norm_w, col[c], 1.0f, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[c][i] = w[i] * (1.0f + f[c][i]);
            }
        }
    };
    float acc[kSums][C][8];
    auto clear = [&](auto& v) {
#pragma unroll
        for (auto& w : v)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = 0.0f;
    };
    clear(acc[0]);
    clear(acc[1]);
    clear(acc[2]);
    struct Rows {
        Raw8<T> dout[R][C], dh[R][C], out[R][C], y[R][C];
    };
    auto load = [&](Rows& q, int64_t at, int64_t stride, int64_t end) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = min(at + r * stride, end - 1);
            const int64_t o = row * D;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if constexpr (kNorm) {
                    q.dh[r][c] = fetch8(dh + o, col[c]);
                    q.out[r][c] = fetch8(out + o, col[c]);
                }
                if (dout) q.dout[r][c] = fetch8(dout + o, col[c]);
                if (y) q.y[r][c] = fetch8(y + o, col[c]);
            }
        }
    };
    int turn = 0;
    // (rows as in block_seam_kernel)
    auto step = [&](Rows& q, int64_t at, int64_t stride, int64_t end, bool busy) {
        float s[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i] = 0.0f;
        auto widen = [&](const Raw8<T>& raw, bool there, float* o) {
            if (there) {
                widen8(raw, o);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = 0.0f;
            }
        };
        if constexpr (N > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    float vo[8], vh[8], vy[8], vd[8], m[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) m[i] = 0.0f;
                    if constexpr (kNorm) {
                        widen8(q.dh[r][c], vh);
                        widen8(q.out[r][c], vo);
                    }
                    if constexpr (kPost) {
                        widen8(q.y[r][c], vy);
                        widen(q.dout[r][c], dout != nullptr, vd);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (kNorm) {
                            vh[i] *= f[c][i];
                            m[0] += vo[i] * vo[i];
                            m[1] += vh[i] * vo[i];
                        }
                        if constexpr (kPost) {
                            constexpr int k = kNorm ? 2 : 0;
                            m[k] += vy[i] * vy[i];
                            const float uy = u[c][i] * vy[i];
                            m[k + 1] += uy * vd[i];
                            if constexpr (kNorm) {
                                m[k + 2] += uy * vh[i];
                                m[k + 3] += uy * vo[i];
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) s[r * N + i] += live[c] ? m[i] : 0.0f;
                }
            }
            row_sums<L>(s, s_part, turn++, W / kWave);
        }
#ifdef V_RENEW
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                renew(q.dout[r][c]);
                if constexpr (kNorm) {
                    renew(q.dh[r][c]);
                    renew(q.out[r][c]);
                }
                renew(q.y[r][c]);
            }
#endif
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float* m = s + r * N;
            const bool on = busy && at + r * stride < end;
            float rr = 0.0f, k1 = 0.0f, ry = 1.0f, k2 = 0.0f;
            if constexpr (kNorm) {
                rr = rsqrtf(m[0] * inv_d + a.eps);
                k1 = rr * rr * rr * (m[1] * inv_d);  // of out in d
            }
            if constexpr (kPost) {
                constexpr int k = kNorm ? 2 : 0;
                ry = rsqrtf(m[k] * inv_d + a.eps);
                float dot = m[k + 1];
                if constexpr (kNorm) dot += rr * m[k + 2] - k1 * m[k + 3];
                k2 = ry * ry * ry * (dot * inv_d);   // of y in dy
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int64_t o = min(at + r * stride, end - 1) * D;
                float d[8], v[8];
                widen(q.dout[r][c], dout != nullptr, d);
                if constexpr (kNorm) {
                    float vo[8], vh[8];
                    widen8(q.dh[r][c], vh);
                    widen8(q.out[r][c], vo);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (on) acc[0][c][i] += vh[i];
                        if (on) acc[1][c][i] += (rr * vh[i]) * vo[i];
                        d[i] += rr * (vh[i] * f[c][i]) - k1 * vo[i];
                    }
                }
                if (y) {
                    float vy[8], w[8];
                    widen8(q.y[r][c], vy);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (on) acc[2][c][i] += d[i] * (ry * vy[i]);
                        w[i] = ry * (u[c][i] * d[i]);
                        if constexpr (kPost) w[i] -= k2 * vy[i];
                    }
                    if (dy && on && live[c]) put8(dy + o, col[c], w);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = a.alpha * d[i];
                if (dx && on && live[c]) put8(dx + o, col[c], v);
            }
        }
    };
    // The parameters' gradients of sequence b from its sums.
    auto finish = [&](int64_t b, const float (&s)[kSums][C][8]) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!live[c]) continue;
            const int64_t o = b * D + col[c];
            float w[8], v[8];
            params8(a.norm_w, col[c], 1.0f, w);
            if (a.dshift) put8(a.dshift + o, s[0][c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[i] * s[1][c][i];
            if (a.dscale) put8(a.dscale + o, v);
            params8(kPost ? a.post_w : nullptr, col[c], 1.0f, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[i] * s[2][c][i];
            if (a.dgate) put8(a.dgate + o, v);
        }
    };
    // The groups' values of the columns added up, in the first group's lanes: by
    // eights, every group's in LDS, in the groups' order.
    auto over_groups = [&](float (&v)[C][8]) {
        if (G == 1) return;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) s_v[i * kSeamThreads + threadIdx.x] = v[c][i];
            __syncthreads();
            if (g == 0)
                for (int o = 1; o < G; ++o)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[c][i] += s_v[i * kSeamThreads + o * W + t];
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
            params(b);
            for (int64_t s = 0; s < a.seq; s += R) {
                Rows q;
                load(q, b * a.seq + s, 1, (b + 1) * a.seq);
                step(q, b * a.seq + s, 1, (b + 1) * a.seq, busy);
            }
            if (busy) finish(b, acc);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float sc[8], gt[8];
                params8(a.scale, b * D + col[c], 0.0f, sc);
                params8(a.gate, b * D + col[c], 1.0f, gt);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    gain[0][c][i] += (1.0f + sc[i]) * acc[1][c][i];  // (zero where not busy)
                    gain[1][c][i] += gt[i] * acc[2][c][i];
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
    params(b);
    if constexpr (V_PRE && C == 1) {
        // the next step's rows are on their way during this one
        Rows q;
        load(q, first + g, G, end);
        for (int64_t at = first; at < end; at += (int64_t)G * R) {
            Rows next;
            load(next, at + (int64_t)G * R + g, G, end);
            step(q, at + g, G, end, true);
            q = next;
        }
    } else {
        for (int64_t at = first; at < end; at += (int64_t)G * R) {
            Rows q;
            load(q, at + g, G, end);
            step(q, at + g, G, end, true);
        }
    }
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

// Adds up the blocks' sums.  A block takes 64 columns (16 threads of four each) of one
// sequence and one of its sums, blockIdx.z; 16 slices of the parts are added in LDS.
//  parts > 0: sums [n][parts][3][D] of n sequences: dshift, dscale, dgate, and per
//             sequence the gains' shares into `gains` [n][2][D] (n = 1: the gains' gradients)
//  parts = 0: gains [n][2][D] into dnorm_w and dpost_w
constexpr int kSumSlices = 16;
__global__ __launch_bounds__(256) void seam_sums_kernel(BlockSeamBackwardArgs a, const float* sums, int64_t n,
                                                        int64_t parts, float* gains) {
    __shared__ float4 s_v[kSumSlices][16];
    const int q = threadIdx.x & 15, slice = threadIdx.x >> 4;
    const int col = blockIdx.x * 64 + q * 4;
    const bool live = col < a.D;
    const int64_t D = a.D, b = blockIdx.y;
    const int k = blockIdx.z, per = parts ? kSums : 2;
    const int64_t m = parts ? parts : n;
    const float* p = sums + (parts ? b * parts * per * D : 0) + k * D + (live ? col : 0);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float4& o) {
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
    };
    constexpr int kFlight = 4;
    int64_t i = slice;
    for (; i + (kFlight - 1) * kSumSlices < m; i += kFlight * kSumSlices) {
        float4 o[kFlight];
#pragma unroll
        for (int j = 0; j < kFlight; ++j)
            o[j] = *reinterpret_cast<const float4*>(p + (i + j * kSumSlices) * per * D);
#pragma unroll
        for (int j = 0; j < kFlight; ++j) add(o[j]);
    }
    for (; i < m; i += kSumSlices) add(*reinterpret_cast<const float4*>(p + i * per * D));
    s_v[slice][q] = v;
    __syncthreads();
    if (slice || !live) return;
    for (int w = 1; w < kSumSlices; ++w) add(s_v[w][q]);
    auto put = [&](float* to, const float* w, float off, const float4& x) {
        const float4 g = w ? *reinterpret_cast<const float4*>(w) : make_float4(1.0f - off, 1.0f - off, 1.0f - off, 1.0f - off);
        *reinterpret_cast<float4*>(to) =
            make_float4((off + g.x) * x.x, (off + g.y) * x.y, (off + g.z) * x.z, (off + g.w) * x.w);
    };
    if (!parts) {
        float* to = k ? a.dpost_w : a.dnorm_w;
        if (to) put(to + col, nullptr, 0.0f, v);
        return;
    }
    const int64_t o = b * D + col;
    if (k == 0) {
        if (a.dshift) put(a.dshift + o, nullptr, 0.0f, v);
        return;
    }
    const bool scale = k == 1;
    if (float* to = scale ? a.dscale : a.dgate)
        put(to + o, scale ? (a.norm_w ? a.norm_w + col : nullptr) : a.post && a.post_w ? a.post_w + col : nullptr, 0.0f,
            v);
    float* to = n > 1 ? gains + (b * 2 + k - 1) * D : scale ? a.dnorm_w : a.dpost_w;
    if (!to) return;
    if (scale) put(to + col, a.scale ? a.scale + o : nullptr, 1.0f, v);
    else put(to + col, a.gate ? a.gate + o : nullptr, 0.0f, v);
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

template <typename T, bool kPost, bool kNorm, int L, int C>
auto grad_kernel(const SeamPlan& p) {
    return p.whole ? seam_grad_kernel<T, kPost, kNorm, true, L, C> : seam_grad_kernel<T, kPost, kNorm, false, L, C>;
}

template <typename T>
hipError_t launch_grad_t(const BlockSeamBackwardArgs& a, hipStream_t s) {
    const SeamPlan p = grad_plan(a.rows, a.D, a.seq);
    float* sums = static_cast<float*>(a.workspace);
    const bool norm = a.dh != nullptr, post = a.post && a.y;
    const hipError_t e = with_seam_shape(p, [&](auto l, auto c) {
        constexpr int L = decltype(l)::value, C = decltype(c)::value;
        auto kern = post ? (norm ? grad_kernel<T, true, true, L, C>(p) : grad_kernel<T, true, false, L, C>(p))
                         : (norm ? grad_kernel<T, false, true, L, C>(p) : grad_kernel<T, false, false, L, C>(p));
        launch_kernel(kern, dim3((unsigned)p.blocks), dim3(p.row_threads * p.groups), 0, s, a, p, sums);
        return hipGetLastError();
    });
    if (e != hipSuccess || !(a.dgate || a.dshift || a.dscale || a.dnorm_w || a.dpost_w)) return e;
    const int64_t n = a.rows / a.seq;
    const unsigned cols = (unsigned)((a.D + 63) / 64);
    float* gains = sums;
    int64_t ng = p.blocks;
    if (!p.whole) {
        gains = sums + p.blocks * kSums * a.D;
        ng = n;
        launch_kernel(seam_sums_kernel, dim3(cols, (unsigned)n, kSums), dim3(256), 0, s, a, (const float*)sums, n,
                      p.parts, gains);
    }
    if ((p.whole || n > 1) && (a.dnorm_w || a.dpost_w))
        launch_kernel(seam_sums_kernel, dim3(cols, 1, 2), dim3(256), 0, s, a, (const float*)gains, ng, (int64_t)0,
                      (float*)nullptr);
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
