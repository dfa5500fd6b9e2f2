// Routing to experts from a router's logits, its gradient, and the intake of a
// routing that the caller has.
//
//   s = softmax(l) or sigmoid(l);  key = s + bias
//   the best top_groups of the groups by the sum of their group_top largest keys,
//   the k largest keys of those groups, ties to the lowest index
//   w_i = scale * s_i / (sum over the chosen + eps), or scale * s_i
//
// An expert whose logit is -inf is masked: its score is zero and it is never
// chosen; slots that stay empty hold -1 with weight zero.  A row's experts are
// written in ascending order.
//
// A wave takes a row; scores and keys are f64, so that the choice is that of
// the definition down to differences of 1e-15.
#include <algorithm>

#include "kernels.hpp"

namespace nomas {

namespace {

constexpr int kRouteThreads = 256;
constexpr int kRouteWaves = kRouteThreads / kWave;

__device__ __forceinline__ double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ double wave_max(double v) {
    for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o));
    return v;
}

// Scores of a row, expert lane + 64 j in s[j]; masked[j] where the logit is -inf
// or there is no such expert.
template <typename T, int V>
__device__ void row_scores(const T* l, int E, int sigmoid, double* raw, double* s) {
    const int lane = threadIdx.x & 63;
    double m = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane + 64 * j;
        raw[j] = e < E ? (double)Elt<T>::to_f32(l[e]) : -INFINITY;
        m = fmax(m, raw[j]);
    }
    double z = 0.0;
    if (!sigmoid) m = wave_max(m);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (raw[j] == -INFINITY) s[j] = 0.0;
        else if (sigmoid) s[j] = 1.0 / (1.0 + exp(-raw[j]));
        else z += s[j] = exp(raw[j] - m);
    }
    if (sigmoid) return;
    z = wave_sum(z);
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (raw[j] != -INFINITY) s[j] /= z;
}

// The wave's largest key and its lowest expert; -1 where every key is -inf.
template <int V>
__device__ int best_of(const double* key, double* best) {
    const int lane = threadIdx.x & 63;
    double b = -INFINITY;
    int at = 1 << 30;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (key[j] > b) {
            b = key[j];
            at = lane + 64 * j;
        }
    for (int o = 32; o; o >>= 1) {
        const double ob = __shfl_xor(b, o);
        const int oa = __shfl_xor(at, o);
        if (ob > b || (ob == b && oa < at)) {
            b = ob;
            at = oa;
        }
    }
    *best = b;
    return b == -INFINITY ? -1 : at;
}

template <typename T, int V>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(RouteArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kRouteWaves + (threadIdx.x >> 6);
    if (blockIdx.x == 0 && a.counts)  // added up by count_kernel
        for (int e = threadIdx.x; e < a.E; e += kRouteThreads) a.counts[e] = 0;
    if (row >= a.rows) return;
    const int E = a.E, k = a.k;
    double raw[V], s[V], key[V];
    row_scores<T, V>(static_cast<const T*>(a.logits) + row * E, E, a.sigmoid, raw, s);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane + 64 * j;
        double q = a.bias && e < E ? s[j] + (double)a.bias[e] : a.groups > 1 ? s[j] : raw[j];
        if (q != q) q = INFINITY;
        key[j] = raw[j] == -INFINITY ? -INFINITY : q;
    }
    if (a.groups > 1) {
        const int per = E / a.groups;
        double score = -INFINITY;  // of group `lane`
        for (int g = 0; g < a.groups; ++g) {
            double in[V], b1, b2 = -INFINITY;
#pragma unroll
            for (int j = 0; j < V; ++j) in[j] = (lane + 64 * j) / per == g ? key[j] : -INFINITY;
            const int at = best_of<V>(in, &b1);
            if (a.group_top > 1 && at >= 0) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (lane + 64 * j == at) in[j] = -INFINITY;
                if (best_of<V>(in, &b2) >= 0) b1 += b2;
            }
            if (lane == g) score = b1;
        }
        uint64_t kept = 0;
        for (int t = 0; t < a.top_groups; ++t) {
            double b;
            const int g = best_of<1>(&score, &b);
            if (g < 0) break;
            kept |= 1ull << g;
            if (lane == g) score = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int g = (lane + 64 * j) / per;
            if (g >= a.groups || !((kept >> g) & 1)) key[j] = -INFINITY;
        }
    }
    unsigned chosen = 0;
    double total = 0.0;
    for (int t = 0; t < k; ++t) {
        double b;
        const int at = best_of<V>(key, &b);
        if (at < 0) break;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (lane + 64 * j == at) {
                key[j] = -INFINITY;
                chosen |= 1u << j;
                total += s[j];
            }
    }
    total = wave_sum(total) + a.eps;
    int n = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const bool in = (chosen >> j) & 1;
        const uint64_t set = __ballot(in);
        if (in) {
            const int at = n + __popcll(set & ((1ull << lane) - 1));
            a.idx[row * k + at] = lane + 64 * j;
            a.w[row * k + at] = (float)(a.scale * (a.renormalize ? s[j] / total : s[j]));
        }
        n += __popcll(set);
    }
    for (int t = n + lane; t < k; t += 64) {
        a.idx[row * k + t] = -1;
        a.w[row * k + t] = 0.0f;
    }
}

constexpr int kCountThreads = 256;

// counts[e] += rows that chose e: a histogram per block in LDS, added with
// integer atomics (their order changes nothing).
__global__ __launch_bounds__(kCountThreads) void count_kernel(const int32_t* idx, int64_t n, int E,
                                                              int32_t* counts) {
    __shared__ int s_n[kMaxRouteExperts];
    for (int e = threadIdx.x; e < E; e += kCountThreads) s_n[e] = 0;
    __syncthreads();
    for (int64_t i = (int64_t)blockIdx.x * kCountThreads + threadIdx.x; i < n;
         i += (int64_t)gridDim.x * kCountThreads)
        if (idx[i] >= 0) atomicAdd(&s_n[idx[i]], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kCountThreads)
        if (s_n[e]) atomicAdd(&counts[e], s_n[e]);
}

template <typename T, int V>
__global__ __launch_bounds__(kRouteThreads) void route_backward_kernel(RouteBackwardArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kRouteWaves + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    const int E = a.E, k = a.k;
    double raw[V], s[V], ds[V];
    row_scores<T, V>(static_cast<const T*>(a.logits) + row * E, E, a.sigmoid, raw, s);
#pragma unroll
    for (int j = 0; j < V; ++j) ds[j] = 0.0;
    // the chosen scores' sum, and their sum weighed by dw
    double total = 0.0, dot = 0.0;
    for (int t = 0; t < k; ++t) {
        const int e = a.idx[row * k + t];
        const double d = a.dw[row * k + t];
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (lane + 64 * j == e && e < E) {
                total += s[j];
                dot += d * s[j];
                ds[j] += d;
            }
    }
    total = wave_sum(total) + a.eps;
    dot = wave_sum(dot);
    // ds_i = scale (dw_i - dot / total) / total for the chosen; the softmax's
    // inner product sum_j s_j ds_j is then scale dot eps / total^2
    const double mean = a.renormalize ? dot / total : 0.0;
    const double up = a.renormalize ? a.scale / total : a.scale;
    const double inner = a.sigmoid ? 0.0 : a.renormalize ? up * mean * a.eps : up * dot;
    for (int t = 0; t < k; ++t) {
        const int e = a.idx[row * k + t];
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (lane + 64 * j == e && e < E) ds[j] -= mean;
    }
    T* out = static_cast<T*>(a.dlogits) + row * E;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane + 64 * j;
        if (e >= E) continue;
        const double d = up * ds[j] - inner;
        const double r = raw[j] == -INFINITY ? 0.0 : a.sigmoid ? d * s[j] * (1.0 - s[j]) : d * s[j];
        out[e] = Elt<T>::from_f32((float)r);
    }
}

// The routing of the caller in the form that the router leaves for the
// dispatch: per row distinct experts in ascending order, then -1; an expert
// outside 0 .. E - 1 is no expert, one named twice has the sum of its weights.
// One block per 64-row chunk, whose histogram it writes.
__global__ __launch_bounds__(kRouteThreads) void given_kernel(GivenRoutingArgs a) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    const int k = a.k, ks = a.k_slots, n = kRouterRows * k;
    int* s_e = reinterpret_cast<int*>(s_raw);           // [64 k] expert, -1 where none or named before
    float* s_w = reinterpret_cast<float*>(s_e + n);     // [64 k]
    int* s_hist = reinterpret_cast<int*>(s_w + n);      // [E_cols]
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * kRouterRows;
    const int nrows = (int)min<int64_t>(kRouterRows, a.rows - row0);
    for (int e = tid; e < a.E_cols; e += kRouteThreads) s_hist[e] = 0;
    for (int i = tid; i < nrows * k; i += kRouteThreads) {
        const int e = a.in_idx[row0 * k + i];
        s_e[i] = e >= 0 && e < a.E ? e : -1;
        s_w[i] = a.in_w[row0 * k + i];
    }
    __syncthreads();
    for (int i = tid; i < nrows * k; i += kRouteThreads) {
        const int r = i / k, e = s_e[i];
        const int* re = s_e + r * k;
        if (e < 0) continue;
        // its place: distinct experts below it; a later mention adds its weight
        int at = 0;
        bool first = true;
        float w = 0.0f;
        for (int t = 0; t < k; ++t) {
            if (re[t] == e) {
                if (r * k + t < i) first = false;
                w += s_w[r * k + t];
            } else if (re[t] >= 0 && re[t] < e) {
                bool again = false;
                for (int u = 0; u < t; ++u) again |= re[u] == re[t];
                at += !again;
            }
        }
        if (!first) continue;
        a.idx[(row0 + r) * ks + at] = e;
        a.w[(row0 + r) * ks + at] = w;
        atomicAdd(&s_hist[e], 1);
    }
    // the empty slots (the dense slot, where there is one, comes last of those taken)
    for (int r = tid; r < nrows; r += kRouteThreads) {
        int live = 0;
        for (int t = 0; t < k; ++t) {
            bool again = s_e[r * k + t] < 0;
            for (int u = 0; u < t; ++u) again |= s_e[r * k + u] == s_e[r * k + t];
            live += !again;
        }
        const int64_t o = (row0 + r) * ks;
        if (ks > k) {
            a.idx[o + live] = a.E;
            a.w[o + live] = a.dense_coef;
            ++live;
            atomicAdd(&s_hist[a.E], 1);
        }
        for (int t = live; t < ks; ++t) {
            a.idx[o + t] = -1;
            a.w[o + t] = 0.0f;
            a.pos[o + t] = -1;
        }
        a.gap[row0 + r] = INFINITY;
    }
    __syncthreads();
    for (int e = tid; e < a.E_cols; e += kRouteThreads)
        a.chunk_counts[(int64_t)blockIdx.x * a.E_cols + e] = s_hist[e];
}

// Calls f with the number of values that a lane holds of E experts.
template <typename F>
hipError_t with_values(int E, F f) {
    if (E <= 64) return f(std::integral_constant<int, 1>{});
    if (E <= 128) return f(std::integral_constant<int, 2>{});
    if (E <= 256) return f(std::integral_constant<int, 4>{});
    if (E <= 512) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 16>{});
}

template <typename T>
hipError_t launch_route_t(const RouteArgs& a, hipStream_t s) {
    const int64_t nblk = std::max<int64_t>(1, (a.rows + kRouteWaves - 1) / kRouteWaves);
    if (nblk > 0x7fffffff) return hipErrorInvalidValue;
    const hipError_t e = with_values(a.E, [&](auto v) {
        launch_kernel(route_kernel<T, decltype(v)::value>, dim3((unsigned)nblk), dim3(kRouteThreads), 0, s, a);
        return hipGetLastError();
    });
    if (e != hipSuccess || !a.counts || a.rows == 0) return e;
    const int64_t n = a.rows * a.k;
    launch_kernel(count_kernel, dim3((unsigned)std::min<int64_t>(64, (n + 1023) / 1024)), dim3(kCountThreads), 0,
                  s, (const int32_t*)a.idx, n, a.E, a.counts);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_route_backward_t(const RouteBackwardArgs& a, hipStream_t s) {
    const int64_t nblk = (a.rows + kRouteWaves - 1) / kRouteWaves;
    if (nblk > 0x7fffffff) return hipErrorInvalidValue;
    return with_values(a.E, [&](auto v) {
        launch_kernel(route_backward_kernel<T, decltype(v)::value>, dim3((unsigned)nblk), dim3(kRouteThreads), 0,
                      s, a);
        return hipGetLastError();
    });
}

}  // namespace

hipError_t launch_route(DType dt, const RouteArgs& a, hipStream_t s) {
    if (a.rows < 0 || a.E < 1 || a.E > kMaxRouteExperts || a.k < 1 || a.k > a.E || a.groups < 1 ||
        a.groups > kMaxRouteGroups || a.E % a.groups != 0)
        return hipErrorInvalidValue;
    switch (dt) {
        case DType::F32: return launch_route_t<float>(a, s);
        case DType::BF16: return launch_route_t<__bf16>(a, s);
        case DType::F16: return launch_route_t<_Float16>(a, s);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_route_backward(DType dt, const RouteBackwardArgs& a, hipStream_t s) {
    if (a.rows < 1 || a.E < 1 || a.E > kMaxRouteExperts || a.k < 1 || a.k > a.E) return hipErrorInvalidValue;
    switch (dt) {
        case DType::F32: return launch_route_backward_t<float>(a, s);
        case DType::BF16: return launch_route_backward_t<__bf16>(a, s);
        case DType::F16: return launch_route_backward_t<_Float16>(a, s);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_given_routing(const GivenRoutingArgs& a, hipStream_t s) {
    const size_t lds = (size_t)kRouterRows * a.k * 8 + (size_t)a.E_cols * 4;
    if (a.rows < 1 || a.k < 1 || a.k > a.E || lds > 160 * 1024) return hipErrorInvalidValue;
    const hipError_t e = hipFuncSetAttribute((const void*)given_kernel,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    launch_kernel(given_kernel, dim3((unsigned)((a.rows + kRouterRows - 1) / kRouterRows)), dim3(kRouteThreads),
                  (uint32_t)lds, s, a);
    return hipGetLastError();
}

}  // namespace nomas
