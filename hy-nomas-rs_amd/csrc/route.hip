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
// The logits are read once and little is written: HBM would take 7 us for 32,768
// rows of 256 f32.  What costs is the choice itself, so it is made for several
// rows by one wave: L = 8 to 64 lanes take a row, each V = 1 to 32 neighbouring
// experts of one group, so that order by lane is order by index.
//  - The k-th largest key is found by bisection of the keys' bits, between the
//    smallest of the lanes' maxima and the largest: each step counts the keys
//    at or above the middle (two instructions a key) and most rows need five to
//    eight steps.
//  - Keys are f32, the definition's choice is made in 64 bits: where a key lies so
//    near the border (of the experts, or of the groups) that its f32 error could
//    carry it across, or a logit is NaN or +inf, the wave decides the row again in
//    f64 (exact_row).  Without bias and groups the keys are the logits themselves:
//    nothing is near, and ties are exact.
//  - The chosen indices meet in LDS, and lane t of a row makes the weight of slot t.
#include <algorithm>
#include <climits>

#include "kernels.hpp"

namespace nomas {

namespace {

constexpr int kRouteThreads = 256;
constexpr int kRouteWaves = kRouteThreads / kWave;
// Blocks of a call that fills the chip (their rows are a loop, so that the bias is
// loaded once and the histogram flushed once)
constexpr int64_t kRouteBlocks = 1024;

__device__ __forceinline__ double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ double wave_max(double v) {
    for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o));
    return v;
}

// ---- the choice in 64 bits, a wave a row ----------------------------------------

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

// Writes a row's choice to `to` (ascending) and returns how many there are; lane
// holds the experts lane, lane + 64, ...
struct ExactRow {
    const float* bias;
    int E, k, sigmoid, groups, top_groups, group_top;
};
template <typename T, int V>
__device__ __noinline__ int exact_row(ExactRow a, const T* l, int* to) {
    const int lane = threadIdx.x & 63, E = a.E;
    double raw[V], key[V];
    double m = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane + 64 * j;
        raw[j] = e < E ? (double)Elt<T>::to_f32(l[e]) : -INFINITY;
        m = fmax(m, raw[j]);
    }
    const bool scores = a.bias || a.groups > 1;
    double z = 0.0;
    if (scores && !a.sigmoid) m = wave_max(m);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (raw[j] == -INFINITY) key[j] = 0.0;
        else if (!scores) key[j] = raw[j];
        else if (a.sigmoid) key[j] = 1.0 / (1.0 + exp(-raw[j]));
        else z += key[j] = exp(raw[j] - m);
    }
    if (scores && !a.sigmoid) z = wave_sum(z);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane + 64 * j;
        if (scores && !a.sigmoid) key[j] /= z;
        if (a.bias && e < E) key[j] += (double)a.bias[e];
        if (key[j] != key[j]) key[j] = INFINITY;
        if (raw[j] == -INFINITY) key[j] = -INFINITY;
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
    for (int t = 0; t < a.k; ++t) {
        double b;
        const int at = best_of<V>(key, &b);
        if (at < 0) break;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (lane + 64 * j == at) {
                key[j] = -INFINITY;
                chosen |= 1u << j;
            }
    }
    int n = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const bool in = (chosen >> j) & 1;
        const uint64_t set = __ballot(in);
        if (in) to[n + __popcll(set & ((1ull << lane) - 1))] = lane + 64 * j;
        n += __popcll(set);
    }
    return n;
}

// ---- sums, extremes and scans over a row's L neighbouring lanes ------------------

template <int kCtrl>
__device__ __forceinline__ int dpp_mov(int v, int old) {
    return __builtin_amdgcn_update_dpp(old, v, kCtrl, 0xf, 0xf, false);
}
// Combines each lane's v with those of the other lanes of its row, by `f`, in all of them.
template <int L, typename F>
__device__ __forceinline__ int over_lanes(int v, F f) {
    static_assert(L >= 8, "lanes of a row");
    v = f(v, dpp_mov<0xb1>(v, v));     // lane ^ 1
    v = f(v, dpp_mov<0x4e>(v, v));     // lane ^ 2
    v = f(v, dpp_mov<0x141>(v, v));    // the other four of eight
    if constexpr (L >= 16) v = f(v, dpp_mov<0x140>(v, v));  // the other eight of sixteen
    if constexpr (L >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
        v = f((int)s[0], (int)s[1]);
    }
    if constexpr (L >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
        v = f((int)s[0], (int)s[1]);
    }
    return v;
}
template <int L>
__device__ __forceinline__ int lanes_add(int v) {
    return over_lanes<L>(v, [](int a, int b) { return a + b; });
}
template <int L>
__device__ __forceinline__ int lanes_min(int v) {
    return over_lanes<L>(v, [](int a, int b) { return min(a, b); });
}
template <int L>
__device__ __forceinline__ int lanes_max(int v) {
    return over_lanes<L>(v, [](int a, int b) { return max(a, b); });
}
template <int L>
__device__ __forceinline__ float lanes_addf(float v) {
    return __int_as_float(over_lanes<L>(__float_as_int(v), [](int a, int b) {
        return __float_as_int(__int_as_float(a) + __int_as_float(b));
    }));
}
template <int L>
__device__ __forceinline__ float lanes_maxf(float v) {
    return __int_as_float(over_lanes<L>(__float_as_int(v), [](int a, int b) {
        return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
    }));
}
template <int L>
__device__ __forceinline__ double lanes_addd(double v) {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Floats in the order of their values as integers (-inf first), and back.
__device__ __forceinline__ int ordered(float v) {
    const int b = __float_as_int(v);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int b) { return __int_as_float(b ^ ((b >> 31) & 0x7fffffff)); }

constexpr int kMasked = (int)0x807fffff;  // ordered(-inf)

// How a row lies on its lanes: of `lanes` for each group (groups rounded up to a
// power of two), lane p of group g holds the experts g per + p each .. + each - 1.
struct RouteShape {
    int L, V;         // lanes of a row, values that a lane may hold
    int lanes, each;  // lanes of a group, experts of a lane
    int per;          // experts of a group
    int vector;       // each == V, whole groups, rows and bias at multiples of V elements: vector loads
};

// V values of consecutive elements, f32.
template <typename T, int V>
__device__ __forceinline__ void load_values(const T* p, float* v) {
    constexpr int bytes = V * (int)sizeof(T), step = bytes < 16 ? bytes : 16, n = step / (int)sizeof(T);
    typedef T Piece __attribute__((ext_vector_type(n > 1 ? n : 2)));
#pragma unroll
    for (int i = 0; i < V; i += n) {
        if constexpr (n == 1) {
            v[i] = Elt<T>::to_f32(p[i]);
        } else {
            const Piece q = *reinterpret_cast<const Piece*>(p + i);
#pragma unroll
            for (int j = 0; j < n; ++j) v[i + j] = Elt<T>::to_f32(q[j]);
        }
    }
}

__global__ void zero_counts_kernel(int32_t* counts, int E) {
    for (int e = threadIdx.x; e < E; e += blockDim.x) counts[e] = 0;
}

// kKeys: the keys are scores (bias or groups); else the logits.
template <typename T, int L, int V, bool kKeys>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(RouteArgs a, RouteShape sh, int direct_counts) {
    constexpr int kRows = kWave / L;  // rows of a wave at a time
    extern __shared__ int s_mem[];
    const int E = a.E, k = a.k;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, p = lane % L, sub = lane / L;
    int* s_idx = s_mem + (wave * kRows + sub) * k;       // this row's choice
    int* s_hist = s_mem + kRouteWaves * kRows * k;       // [E]
    if (a.counts) {
        for (int e = threadIdx.x; e < E; e += kRouteThreads) s_hist[e] = 0;
        __syncthreads();
    }
    const int g = p / sh.lanes, at0 = (p - g * sh.lanes) * sh.each;
    const bool in_group = g < a.groups;
    const int first = in_group ? g * sh.per + at0 : 0;      // the lane's experts: first .. first + n - 1
    const int n = in_group ? max(0, min(sh.each, sh.per - at0)) : 0;
    const T* logits = static_cast<const T*>(a.logits);
    float bias[V];
    if constexpr (kKeys) {
#pragma unroll
        for (int j = 0; j < V; ++j) bias[j] = a.bias && j < n ? a.bias[first + j] : 0.0f;
    }
    // (a NaN or infinite bias: every row is decided in exact_row)
    bool odd_bias = false;
    if constexpr (kKeys) {
#pragma unroll
        for (int j = 0; j < V; ++j) odd_bias |= !(fabsf(bias[j]) < INFINITY);
    }
    const ExactRow exact_args = {a.bias, E, k, a.sigmoid, a.groups, a.top_groups, a.group_top};
    const int64_t stride = (int64_t)gridDim.x * kRouteWaves * kRows;
    for (int64_t row0 = ((int64_t)blockIdx.x * kRouteWaves + wave) * kRows; row0 < a.rows; row0 += stride) {
        const int64_t row = min(row0 + sub, a.rows - 1);
        const bool real = row0 + sub < a.rows;
        const T* l = logits + row * E;
        float raw[V];
        if (sh.vector) {
            load_values<T, V>(l + first, raw);
            if (!in_group)
#pragma unroll
                for (int j = 0; j < V; ++j) raw[j] = -INFINITY;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) raw[j] = j < n ? Elt<T>::to_f32(l[first + j]) : -INFINITY;
        }
        // +inf and NaN: decided in exact_row
        float top = raw[0], all = raw[0];
#pragma unroll
        for (int j = 1; j < V; ++j) {
            top = fmaxf(top, raw[j]);
            all += raw[j];
        }
        bool odd = odd_bias || all != all || all == INFINITY;
        float zsum = 1.0f;
        if (!a.sigmoid) {
            top = lanes_maxf<L>(top);
            float z = 0.0f;
            const float c = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int j = 0; j < V; ++j) z += __expf(raw[j] - c);
            zsum = lanes_addf<L>(z);
            top = c;
        }
        int key[V];
        float near = 0.0f;  // how far a key may be off
        if constexpr (kKeys) {
            const float zi = 1.0f / zsum;
            near = a.sigmoid ? 0x1p-21f : 0x1p-19f * zi;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + __expf(-raw[j])) : __expf(raw[j] - top) * zi;
                key[j] = ordered(raw[j] == -INFINITY ? -INFINITY : s + bias[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) key[j] = ordered(raw[j]);
        }
        if constexpr (kKeys) {
            if (a.groups > 1) {
                // the group's two largest, over its lanes
                float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float v = unordered(key[j]);
                    m2 = fmaxf(m2, fminf(m1, v));
                    m1 = fmaxf(m1, v);
                }
                for (int o = 1; o < sh.lanes; o <<= 1) {
                    const float o1 = __shfl_xor(m1, o), o2 = __shfl_xor(m2, o);
                    m2 = fmaxf(fmaxf(m2, o2), fminf(m1, o1));
                    m1 = fmaxf(m1, o1);
                }
                const float score = a.group_top > 1 && m2 != -INFINITY ? m1 + m2 : m1;
                int before = 0;  // groups ahead of this one
                float gap = INFINITY;  // to the nearest other group's score on the other side of the border
                for (int q = 0; q < a.groups; ++q) {
                    const float o = __shfl(score, sub * L + q * sh.lanes);
                    before += o > score || (o == score && q < g);
                }
                const bool kept = before < a.top_groups && in_group;
                const float low = -lanes_maxf<L>(kept ? -score : -INFINITY);
                const float high = lanes_maxf<L>(kept || !in_group ? -INFINITY : score);
                gap = low - high;
                odd |= high != -INFINITY && !(gap > 4.0f * (near + 0x1p-22f * fabsf(high)));
#pragma unroll
                for (int j = 0; j < V; ++j) key[j] = kept ? key[j] : kMasked;
            }
        }
        // bisection: count(key >= lo) >= k > count(key >= hi)
        int most = kMasked, least = INT_MAX, live = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            most = max(most, key[j]);
            live += key[j] != kMasked;
        }
        const int lanes_in = lanes_add<L>(most != kMasked);
        const int total = lanes_add<L>(live);
        if (lanes_in >= k) {
            least = most == kMasked ? INT_MAX : most;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) least = min(least, key[j] == kMasked ? INT_MAX : key[j]);
        }
        int lo = lanes_min<L>(least), hi = lanes_max<L>(most);
        bool done = total <= k;      // all of them
        if (done) lo = kMasked + 1;
        else hi = hi < INT_MAX ? hi + 1 : hi;
        bool exact = done;           // count(key >= lo) is what is taken
        // (32 steps halve any bracket to nothing; rows with a NaN may not end before)
        for (int i = 0; i < 33 && __ballot(!done); ++i) {
            // (lo + hi) / 2 without overflow, towards lo
            const int mid = (lo & hi) + ((lo ^ hi) >> 1);
            int c = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) c += key[j] >= mid;
            c = lanes_add<L>(c);
            if (!done) {
                if (mid == lo) {     // lo is the k-th key, and there are more of it than places
                    done = true;
                } else if (c == k) {
                    lo = mid;
                    done = exact = true;
                } else if (c > k) {
                    lo = mid;
                } else {
                    hi = mid;
                }
            }
        }
        unsigned chosen = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) chosen |= (unsigned)(key[j] >= lo) << j;
        if constexpr (kKeys) {
            if (total > k) {
                const float border = unordered(lo);
                float gap = INFINITY;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    gap = fminf(gap, fabsf(unordered(key[j]) - border));
                odd |= !exact || !(gap > near + 0x1p-22f * fabsf(border));
            }
        } else if (__ballot(!exact)) {
            // of the experts at lo the first, in index order, for the places that are left
            unsigned ties = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) ties |= (unsigned)(key[j] == lo) << j;
            const int above = lanes_add<L>(__popc(chosen & ~ties));
            int before = __popc(ties);
            const int own = before;
#pragma unroll
            for (int o = 1; o < L; o <<= 1) {
                const int t = __shfl_up(before, o, L);
                if (p >= o) before += t;
            }
            int room = k - above - (before - own);
            unsigned take = 0;
            for (unsigned m = ties; m && room > 0; m &= m - 1, --room) take |= m & -m;
            if (!exact) chosen = (chosen & ~ties) | take;
        }
        int before = __popc(chosen);
        const int own = before;
#pragma unroll
        for (int o = 1; o < L; o <<= 1) {
            const int t = __shfl_up(before, o, L);
            if (p >= o) before += t;
        }
        int found = __shfl(before, sub * L + L - 1);
        before -= own;
        for (unsigned m = chosen; m; m &= m - 1, ++before)
            if (before < k) s_idx[before] = first + __ffs(m) - 1;
        uint64_t again = __ballot(odd && real);
        while (again) {  // (the same for the whole wave)
            const int r = __builtin_ctzll(again) / L;
            again &= ~((L < 64 ? (1ull << (L & 63)) - 1 : ~0ull) << (r * L));
            const int c = exact_row<T, (L * V + 63) / 64>(exact_args, logits + min(row0 + r, a.rows - 1) * E,
                                                           s_mem + (wave * kRows + r) * k);
            if (sub == r) found = c;
        }
        __builtin_amdgcn_wave_barrier();
        found = min(found, k);
        // slot t of the row: its weight, from f64 scores
        double sum = 0.0;
        for (int t0 = 0; t0 < k; t0 += L) {
            const int t = t0 + p;
            if (t < found) {
                const double v = Elt<T>::to_f32(l[s_idx[t]]);
                sum += a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)top) / (double)zsum;
            }
        }
        if (a.renormalize) sum = lanes_addd<L>(sum) + a.eps;
        for (int t0 = 0; t0 < k; t0 += L) {
            const int t = t0 + p;
            if (t >= k || !real) continue;
            int e = -1;
            float w = 0.0f;
            if (t < found) {
                e = s_idx[t];
                const double v = Elt<T>::to_f32(l[e]);
                const double s = a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)top) / (double)zsum;
                w = (float)(a.scale * (a.renormalize ? s / sum : s));
                if (a.counts) atomicAdd(&s_hist[e], 1);
            }
            a.idx[row * k + t] = e;
            a.w[row * k + t] = w;
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (!a.counts) return;
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
        if (direct_counts) a.counts[e] = s_hist[e];
        else if (s_hist[e]) atomicAdd(&a.counts[e], s_hist[e]);  // (integers: in any order)
    }
}

// Lanes and values: the fewest lanes that hold a row with at most 16 values each,
// each group on lanes of its own.
RouteShape route_shape(int E, int groups) {
    RouteShape s{};
    int gp = 1;
    while (gp < groups) gp <<= 1;
    s.per = E / groups;
    for (s.L = std::max(8, gp);; s.L <<= 1) {
        s.lanes = s.L / gp;
        s.each = (s.per + s.lanes - 1) / s.lanes;
        if (s.each <= 16 || s.L == kWave) break;
    }
    for (s.V = 1; s.V < s.each; s.V <<= 1) {}
    return s;
}


// ---- the gradient -----------------------------------------------------------------

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

template <typename T, int L, int V>
hipError_t launch_route_shape(const RouteArgs& a, const RouteShape& sh, hipStream_t s) {
    constexpr int rows = kRouteWaves * (kWave / L);
    const int64_t need = (a.rows + rows - 1) / rows;
    const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min(need, kRouteBlocks));
    const uint32_t lds = (uint32_t)(rows * a.k + (a.counts ? a.E : 0)) * 4;
    const int direct = blocks == 1;
    if (a.counts && !direct) launch_kernel(zero_counts_kernel, dim3(1), dim3(256), 0, s, a.counts, a.E);
    auto kern = a.bias || a.groups > 1 ? route_kernel<T, L, V, true> : route_kernel<T, L, V, false>;
    launch_kernel(kern, dim3(blocks), dim3(kRouteThreads), lds, s, a, sh, direct);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_route_t(const RouteArgs& a, hipStream_t s) {
    RouteShape sh = route_shape(a.E, a.groups);
    const uintptr_t at = (uintptr_t)std::min<size_t>(16, sh.V * sizeof(T)) - 1;
    sh.vector = sh.each == sh.V && sh.per == sh.lanes * sh.V && !((uintptr_t)a.logits & at) &&
                !((a.E * sizeof(T)) & at);
    switch (sh.L * 64 + sh.V) {
#define ROUTE_SHAPE(l, v) \
    case l * 64 + v: return launch_route_shape<T, l, v>(a, sh, s);
        ROUTE_SHAPE(8, 1)
        ROUTE_SHAPE(8, 2)
        ROUTE_SHAPE(8, 4)
        ROUTE_SHAPE(8, 8)
        ROUTE_SHAPE(8, 16)
        ROUTE_SHAPE(16, 1)
        ROUTE_SHAPE(16, 2)
        ROUTE_SHAPE(16, 4)
        ROUTE_SHAPE(16, 8)
        ROUTE_SHAPE(16, 16)
        ROUTE_SHAPE(32, 1)
        ROUTE_SHAPE(32, 2)
        ROUTE_SHAPE(32, 4)
        ROUTE_SHAPE(32, 8)
        ROUTE_SHAPE(32, 16)
        ROUTE_SHAPE(64, 1)
        ROUTE_SHAPE(64, 2)
        ROUTE_SHAPE(64, 4)
        ROUTE_SHAPE(64, 8)
        ROUTE_SHAPE(64, 16)
        ROUTE_SHAPE(64, 32)
#undef ROUTE_SHAPE
    }
    return hipErrorInvalidValue;
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
