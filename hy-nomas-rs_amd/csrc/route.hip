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
//  - Each lane keeps its four largest keys in order.  A round takes the largest key over the
//    lanes and shifts the list that it came from: the k-th round's is the border, for up to
//    16 places.  Where that does not count k keys (ties, a lane that holds more of the best than
//    its list) and for longer choices the border is found by bisection of the keys' bits.
//  - Keys are f32, the definition's choice is made in 64 bits: the keys that lie so
//    near the border (of the experts, or of the groups) that their f32 error could
//    carry them across are made again in f64, and decided among themselves.
//    Without bias and groups the keys are the logits: nothing is near, ties are exact.
//  - The chosen indices meet in LDS, and lane t of a row makes the weight of slot t.
//
// 32,768 rows of 256 f32, sigmoid and bias, 8 groups, top-8: 21.5 us (an f64 wave a row: 196).
// Leaving one part out at a time makes it shorter by: the read 7.2, keys 2.5, lists and groups 2,
// rounds 4, choice and weights 4, doubtful rows 2.3 (they overlap somewhat).  The masks of the loads
// that are no vector loads, kept for all rows, push 107 scalar registers into vector ones.  4,744 rows of
// 64 bf16 4.6 us; one row 4.6.  The counts take 3 (4,744 rows) to 4 us more.  Top-24 of the same rows
// (bisection) 37 us; 8,192 rows of 1,000 f32, softmax top-8, 37 us; of 1,020 in 60 groups, 32 values a
// lane at 179 registers, top-32, 91 us.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "kernels.hpp"

namespace nomas {

namespace {

constexpr int kRouteThreads = 256;
constexpr int kRouteWaves = kRouteThreads / kWave;
// Blocks of a call that fills the chip (their rows are a loop, so that the bias is
// loaded once and the histogram flushed once)
constexpr int64_t kRouteBlocks = 1024;
constexpr int64_t kRouteGradBlocks = 8192;
constexpr int64_t kRouteWavesMin = 1024;  // a wave for each SIMD

// ---- sums, extremes and scans over a row's L neighbouring lanes ------------------

// Another lane's v (0 where there is none): in a form that the instruction that uses it
// takes as its operand.
template <int kCtrl>
__device__ __forceinline__ int dpp_mov(int v) {
    return __builtin_amdgcn_update_dpp(0, v, kCtrl, 0xf, 0xf, true);
}
// Combines each lane's v with those of the other lanes of its row, by `f`, in all of them.
template <int L, typename F>
__device__ __forceinline__ int over_lanes(int v, F f) {
    static_assert(L >= 8, "lanes of a row");
    v = f(v, dpp_mov<0xb1>(v));     // lane ^ 1
    v = f(v, dpp_mov<0x4e>(v));     // lane ^ 2
    v = f(v, dpp_mov<0x141>(v));    // the other four of eight
    if constexpr (L >= 16) v = f(v, dpp_mov<0x140>(v));  // the other eight of sixteen
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
// The sum over the row's lanes up to and including this one (p: its place in the row).
template <int L>
__device__ __forceinline__ int lanes_scan(int v, int p) {
#pragma unroll
    for (int o = 1; o < (L < 16 ? L : 16); o <<= 1) {  // row_shr: o
        const int t = o == 1 ? dpp_mov<0x111>(v) : o == 2 ? dpp_mov<0x112>(v) : o == 4 ? dpp_mov<0x114>(v)
                                                                                     : dpp_mov<0x118>(v);
        v += L < 16 && p < o ? 0 : t;
    }
    if constexpr (L >= 32) v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast: 15
    if constexpr (L >= 64) v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast: 31
    return v;
}
// The row's largest (d, lowest index), in all of its lanes.
template <int L>
__device__ __forceinline__ void lanes_best(double& d, int& e) {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) {
        const double od = __shfl_xor(d, o);
        const int oe = __shfl_xor(e, o);
        if (od > d || (od == d && oe < e)) {
            d = od;
            e = oe;
        }
    }
}
template <int L>
__device__ __forceinline__ double lanes_addd(double v) {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// What the wave's lanes have written to LDS is there for all of them: LDS takes a
// wave's operations in order, so this only keeps the compiler from moving them.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Floats in the order of their values as integers (-inf first; not for -0), and back.
__device__ __forceinline__ int ordered(float v) {
    const int b = __float_as_int(v);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int b) { return __int_as_float(b ^ ((b >> 31) & 0x7fffffff)); }

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

// counts[e] += rows that chose e, of n indices: a histogram per block in LDS, added
// with integer atomics (in any order the same).  Few blocks: their atomics meet at the
// same E addresses (1,024 blocks that flush 256 counts each take 12 us).
constexpr int kCountThreads = 1024, kCountBlocks = 32;
__global__ __launch_bounds__(kCountThreads) void route_count_kernel(const int32_t* idx, int64_t n, int E,
                                                                    int32_t* counts) {
    __shared__ int s_n[kMaxRouteExperts];
    for (int e = threadIdx.x; e < E; e += kCountThreads) s_n[e] = 0;
    __syncthreads();
    const int64_t stride = (int64_t)gridDim.x * kCountThreads;
    for (int64_t i = (int64_t)blockIdx.x * kCountThreads + threadIdx.x; i < n; i += 8 * stride) {
        int e[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) e[u] = idx[min(i + u * stride, n - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i + u * stride < n && e[u] >= 0) atomicAdd(&s_n[e[u]], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kCountThreads)
        if (s_n[e]) atomicAdd(&counts[e], s_n[e]);
}

// The keys that the choice goes by, as integers in their order: f32 scores and bias,
// or f32 logits; of 16-bit logits the bits that they have, with the index behind
// them, so that no two are equal.
template <typename T, bool kKeys> struct RouteKey {
    static constexpr int kDrop = 0;  // zero bits of the f32 value
    static constexpr bool kUnique = false;
};
template <> struct RouteKey<__bf16, false> {
    static constexpr int kDrop = 16;
    static constexpr bool kUnique = true;
};
template <> struct RouteKey<_Float16, false> {
    static constexpr int kDrop = 13;
    static constexpr bool kUnique = true;
};
__device__ __forceinline__ int middle(int a, int b, int c) {
    int r;
    asm("v_med3_i32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

constexpr int kRounds = 16;  // the largest top_k whose keys are taken off one by one
constexpr int kList = 4;     // keys that a lane keeps in order for that

// kKeys: the keys are scores (bias or groups); else the logits.
template <typename T, int L, int V, bool kKeys>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(RouteArgs a, RouteShape sh) {
    constexpr int kRows = kWave / L;  // rows of a wave at a time
    constexpr bool kUnique = RouteKey<T, kKeys>::kUnique;
    constexpr int kNone = kUnique ? INT_MIN : (int)0x807fffff;  // masked, or no expert: -inf
    extern __shared__ int s_mem[];
    const int E = a.E, k = a.k;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, p = lane % L, sub = lane / L;
    int* s_idx = s_mem + (wave * kRows + sub) * k;       // this row's choice
    int* s_hist = s_mem + kRouteWaves * kRows * k;       // [E]
    // counts: a single block writes its histogram, others leave it to
    // route_count_kernel, which adds to zeros
    const bool hist = a.counts && gridDim.x == 1;
    if (a.counts && blockIdx.x == 0) {
        for (int e = threadIdx.x; e < E; e += kRouteThreads) (hist ? s_hist : a.counts)[e] = 0;
        if (hist) __syncthreads();
    }
    const int g = p / sh.lanes, at0 = (p - g * sh.lanes) * sh.each;
    const bool in_group = g < a.groups;
    const int first = in_group ? g * sh.per + at0 : 0;      // the lane's experts: first .. first + n - 1
    const int n = in_group ? max(0, min(sh.each, sh.per - at0)) : 0;
    const T* logits = static_cast<const T*>(a.logits);
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
        float bias[V];  // (read again for each row: kept, its registers cost a wave per SIMD)
        if constexpr (kKeys) {
            if (a.bias && sh.vector) {
                load_values<float, V>(a.bias + first, bias);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) bias[j] = a.bias && j < n ? a.bias[first + j] : 0.0f;
            }
        }
        // ---- keys ----
        constexpr float kLog2e = 1.44269504f;
        float top = 0.0f, zsum = 1.0f;  // of the softmax
        if (!a.sigmoid) {
            top = raw[0];
#pragma unroll
            for (int j = 1; j < V; ++j) top = fmaxf(top, raw[j]);
            top = lanes_maxf<L>(top);
            if (top == -INFINITY) top = 0.0f;
            zsum = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) zsum += __builtin_amdgcn_exp2f((raw[j] - top) * kLog2e);
            zsum = lanes_addf<L>(zsum);
        }
        int key[V];
        float near = 0.0f;  // how far a key may be off
        float all = 0.0f;   // a NaN if a key is one
        if constexpr (kKeys) {
            // Errors of s, in half steps of f32: sigmoid, s (1 - s) (1.5 |l| + 2) + 3 s < 4;
            // softmax, times 1 / Z: 2.5 |l - top| exp(l - top) + 2 < 3, and Z's own, at most
            // 2.5 ln E + 2 of its terms and 37 of their sum
            float s[V];
            if (a.sigmoid) {
                near = 0x1p-21f;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    s[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(raw[j] * -kLog2e));
            } else {
                const float zi = 1.0f / zsum;
                near = 0x1p-18f * zi;
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] = __builtin_amdgcn_exp2f((raw[j] - top) * kLog2e) * zi;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s[j] += bias[j];
                all += s[j];
                key[j] = ordered(raw[j] == -INFINITY ? -INFINITY : s[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                all += raw[j];
                key[j] = ordered(raw[j] + 0.0f);  // (-0 is 0)
                if constexpr (kUnique)
                    key[j] = raw[j] == -INFINITY ? kNone
                                                 : (key[j] >> RouteKey<T, kKeys>::kDrop) * kMaxRouteExperts +
                                                       (kMaxRouteExperts - 1 - first - j);
            }
        }
        // a NaN counts as the largest (in a softmax all of the row's scores are NaN then,
        // and after +inf too)
        if (__ballot(all != all)) {
            constexpr int kInf = 0x7f800000 >> RouteKey<T, kKeys>::kDrop;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = kKeys ? unordered(key[j]) : raw[j];
                if (v != v) key[j] = kUnique ? kInf * kMaxRouteExperts + (kMaxRouteExperts - 1 - first - j) : kInf;
            }
        }
        // The key of expert e in 64 bits.
        double z64 = 0.0;
        auto sum64 = [&]() {
            if (a.sigmoid || z64 != 0.0) return;
            for (int j = 0; j < n; ++j) {
                const float v = Elt<T>::to_f32(l[first + j]);
                if (v != -INFINITY) z64 += exp((double)v - (double)top);
            }
            z64 = lanes_addd<L>(z64);
        };
        auto key64 = [&](int e) {
            const double v = Elt<T>::to_f32(l[e]);
            double s = a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)top) / z64;
            if (a.bias) s += (double)a.bias[e];
            return s == s ? s : (double)INFINITY;
        };
        // the lane's largest keys in descending order (in four variables: of an array the
        // compiler makes selections by index, twice the instructions of a round)
        int t0 = kNone, t1 = kNone, t2 = kNone, t3 = kNone;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            t3 = middle(t3, t2, key[j]);
            t2 = middle(t2, t1, key[j]);
            t1 = middle(t1, t0, key[j]);
            t0 = max(t0, key[j]);
        }
        bool kept = in_group;
        if constexpr (kKeys) {
            if (a.groups > 1) {
                // the group's two largest, over its lanes
                int i1 = t0, i2 = t1;
                for (int o = 1; o < sh.lanes; o <<= 1) {
                    const int o1 = __shfl_xor(i1, o), o2 = __shfl_xor(i2, o);
                    i2 = max(max(i2, o2), min(i1, o1));
                    i1 = max(i1, o1);
                }
                // (half of the sum, or of the one that there is: two biases' may pass f32's range)
                const float m1 = unordered(i1), m2 = unordered(i2);
                const float score = a.group_top > 1 && m2 != -INFINITY ? 0.5f * m1 + 0.5f * m2 : 0.5f * m1;
                int ahead = 0;  // groups before this one
                for (int q = 0; q < a.groups; ++q) {
                    const float o = __shfl(score, sub * L + q * sh.lanes);
                    ahead += o > score || (o == score && q < g);
                }
                kept &= ahead < a.top_groups;
                const float low = -lanes_maxf<L>(kept ? -score : -INFINITY);
                const float high = lanes_maxf<L>(kept || !in_group ? -INFINITY : score);
                // two keys' errors on either side; a key's grows with it, not with the sum
                const float size = 0.5f * fabsf(m1) + (m2 == -INFINITY ? 0.0f : 0.5f * fabsf(m2));
                const float most = lanes_maxf<L>(in_group && size < INFINITY ? size : 0.0f);
                const bool doubt =
                    high != -INFINITY && low < INFINITY && !(low - high > 2.0f * near + 0x1p-21f * most);
                if (__ballot(doubt)) {
                    sum64();
                    // those that may be among the group's largest
                    const float last = a.group_top > 1 ? m2 : m1;
                    const float from = last - 2.0f * (near + 0x1p-22f * fabsf(last));
                    double d1 = -INFINITY, d2 = -INFINITY;
                    unsigned may = 0;
#pragma unroll
                    for (int j = 0; j < V; ++j) may |= (unsigned)(key[j] != kNone && !(unordered(key[j]) < from)) << j;
                    if (!doubt) may = 0;
                    for (; may; may &= may - 1) {
                        const double d = key64(first + __ffs(may) - 1);
                        d2 = fmax(d2, fmin(d1, d));
                        d1 = fmax(d1, d);
                    }
                    for (int o = 1; o < sh.lanes; o <<= 1) {
                        const double o1 = __shfl_xor(d1, o), o2 = __shfl_xor(d2, o);
                        d2 = fmax(fmax(d2, o2), fmin(d1, o1));
                        d1 = fmax(d1, o1);
                    }
                    const double exact = a.group_top > 1 && d2 != -INFINITY ? d1 + d2 : d1;
                    ahead = 0;
                    for (int q = 0; q < a.groups; ++q) {
                        const double o = __shfl(exact, sub * L + q * sh.lanes);
                        ahead += o > exact || (o == exact && q < g);
                    }
                    if (doubt) kept = ahead < a.top_groups && in_group;
                }
                if (!kept) {
                    t0 = t1 = t2 = t3 = kNone;
#pragma unroll
                    for (int j = 0; j < V; ++j) key[j] = kNone;
                }
            }
        }
        // ---- the k-th key ----
        int border = kNone;  // chosen: the keys at or above it, but for kNone
        if (k <= kRounds) {
            for (int i = 0; i < k; ++i) {
                border = lanes_max<L>(t0);
                const bool off = t0 == border;
                t0 = off ? t1 : t0;
                t1 = off ? t2 : t1;
                t2 = off ? t3 : t2;
                t3 = off ? kNone : t3;
            }
        }
        auto bits = [&](int from) {  // of the lane's keys at or above `from`
            unsigned m = 0;
#pragma unroll
            for (int j = V - 1; j >= 0; --j) m = m + m + (key[j] >= from);
            return m;
        };
        unsigned chosen = bits(max(border, kNone + 1));
        int own = __popc(chosen);
        int upto = lanes_scan<L>(own, p);
        int found = lanes_max<L>(upto);
        const bool found_it = k <= kRounds && (border == kNone ? found <= k : found == k);
        bool by_index = false;   // the places left go to the first of those with the key `border`
        if (__ballot(!found_it)) {
            // Bisection of the keys' bits: count(key >= lo) >= k > count(key >= hi).  For
            // long choices, ties, and lanes that hold more of the best than their list.
            int most = kNone, least = INT_MAX, live = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                most = max(most, key[j]);
                least = min(least, key[j] == kNone ? INT_MAX : key[j]);
                live += key[j] != kNone;
            }
            live = lanes_add<L>(live);
            int lo = lanes_min<L>(least), hi = lanes_max<L>(most);
            bool done = found_it || live <= k, exact = done;
            if (!found_it) border = kNone;
            if (!done) hi = hi < INT_MAX ? hi + 1 : hi;
            // (32 steps halve any bracket to nothing)
            for (int i = 0; i < 33 && __ballot(!done); ++i) {
                const int mid = (lo & hi) + ((lo ^ hi) >> 1);
                int c = 0;
#pragma unroll
                for (int j = 0; j < V; ++j) c += key[j] >= mid;  // (lo, and so mid, is above kNone)
                c = lanes_add<L>(c);
                if (!done) {
                    if (mid == lo) {  // lo is the k-th key, and there are more of it than places
                        done = true;
                        border = lo;
                    } else if (c == k) {
                        done = exact = true;
                        border = mid;
                    } else if (c > k) {
                        lo = mid;
                    } else {
                        hi = mid;
                    }
                }
            }
            if (!found_it) {
                chosen = bits(max(border, kNone + 1));
                by_index = !exact;
            }
        }
        if constexpr (kKeys) {
            // the largest key that is left out: near the border?
            int next = k <= kRounds ? t0 : kNone;
            if (__ballot(own >= kList || !found_it)) {  // (the list may have ended before it)
#pragma unroll
                for (int j = 0; j < V; ++j) next = max(next, (chosen >> j) & 1 ? kNone : key[j]);
            }
            next = lanes_max<L>(next);
            const float edge = unordered(border);
            const float off = 2.0f * (near + 0x1p-22f * fabsf(edge));
            const bool doubt = border != kNone && edge < INFINITY &&
                               (by_index || (next != kNone && !(edge - unordered(next) > off)));
            if (__ballot(doubt)) {
                unsigned ties = 0, sure = 0;  // the doubtful ones, and those ahead of them
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const bool tie = fabsf(unordered(key[j]) - edge) <= off;
                    ties |= (unsigned)tie << j;
                    sure |= (unsigned)(key[j] > border && !tie) << j;
                }
                if (!doubt) ties = 0;
                int places = doubt ? k - lanes_add<L>(__popc(sure)) : 0;
                // the same logit and bias: a tie in 64 bits too
                int l0 = INT_MAX, l1 = INT_MIN, b0 = INT_MAX, b1 = INT_MIN;
                for (unsigned m = ties; m; m &= m - 1) {
                    const int e = first + __ffs(m) - 1;
                    const int v = ordered(Elt<T>::to_f32(l[e]) + 0.0f), w = a.bias ? ordered(a.bias[e] + 0.0f) : 0;
                    l0 = min(l0, v);
                    l1 = max(l1, v);
                    b0 = min(b0, w);
                    b1 = max(b1, w);
                }
                const bool same = lanes_min<L>(l0) == lanes_max<L>(l1) && lanes_min<L>(b0) == lanes_max<L>(b1);
                if (doubt) chosen = sure;
                if (__ballot(doubt && same)) {
                    const int room = places - (lanes_scan<L>(__popc(ties), p) - __popc(ties));
                    unsigned take = 0;
                    int r = room;
                    for (unsigned m = ties; m && r > 0; m &= m - 1, --r) take |= m & -m;
                    if (doubt && same) {
                        chosen = sure | take;
                        places = 0;
                    }
                }
                if (__ballot(places > 0)) {
                    sum64();
                    unsigned left = places > 0 ? ties : 0;
                    double d = -INFINITY;  // the lane's best of those left
                    int at = INT_MAX;
                    bool again = true;
                    while (__ballot(places > 0)) {
                        if (again) {
                            d = -INFINITY;
                            at = INT_MAX;
                            for (unsigned m = left; m; m &= m - 1) {
                                const int e = first + __ffs(m) - 1;
                                const double v = key64(e);
                                if (v > d) {
                                    d = v;
                                    at = e;
                                }
                            }
                        }
                        double best = d;
                        int e = at;
                        lanes_best<L>(best, e);
                        again = places > 0 && e == at && at != INT_MAX;
                        if (again) {
                            chosen |= 1u << (e - first);
                            left &= ~(1u << (e - first));
                        }
                        --places;
                    }
                }
                if (doubt) by_index = false;
            }
        }
        if (__ballot(by_index)) {
            unsigned ties = 0, sure = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ties |= (unsigned)(key[j] == border) << j;
                sure |= (unsigned)(key[j] > border) << j;
            }
            int room = k - lanes_add<L>(__popc(sure)) - (lanes_scan<L>(__popc(ties), p) - __popc(ties));
            unsigned take = 0;
            for (unsigned m = ties; m && room > 0; m &= m - 1, --room) take |= m & -m;
            if (by_index) chosen = sure | take;
        }
        // ---- the choice, and its weights ----
        own = __popc(chosen);
        upto = lanes_scan<L>(own, p);
        found = lanes_max<L>(upto);
        int place = upto - own;
        for (unsigned m = chosen; m; m &= m - 1, ++place)
            if (place < k) s_idx[place] = first + __ffs(m) - 1;
        wave_sync();
        // lane t of the row: slot t.  Renormalised weights come from scores (and eps) relative to the
        // largest chosen one or eps, whichever is larger: at their own scale all of the chosen may
        // underflow (a softmax whose bias chooses far below the row's largest logit, a sigmoid of
        // low logits), at the scores' eps may overflow.
        float m = 0.0f;  // a softmax's scores are exp(v - top - m), a sigmoid's s exp(-m), m <= 0
        auto score = [&](float v) {
            if (!a.sigmoid) return expf(v - top - m);
            const float q = expf(-fabsf(v));
            return (v < 0.0f ? expf(v - m) : 1.0f) / (1.0f + q);  // (a NaN stays one)
        };
        int e0 = -1;
        float v0 = -INFINITY, most = -INFINITY;
        for (int t = p; t < k; t += L) {
            const int e = t < found ? s_idx[t] : -1;
            const float v = e >= 0 ? Elt<T>::to_f32(l[e]) : -INFINITY;
            if (t < L) {
                e0 = e;
                v0 = v;
            }
            most = fmaxf(most, v);
        }
        float log_eps = 0.0f;
        if (a.renormalize) {
            most = lanes_maxf<L>(most);
            log_eps = a.log_eps + (a.sigmoid ? 0.0f : logf(zsum));
            m = a.sigmoid ? fminf(fmaxf(most, log_eps), 0.0f) : fmaxf(most - top, log_eps);
        }
        float s0 = 0.0f, sum = 0.0f;
        for (int t = p; t < k; t += L) {
            const int e = t < L ? e0 : t < found ? s_idx[t] : -1;
            const float s = e >= 0 ? score(t < L ? v0 : Elt<T>::to_f32(l[e])) : 0.0f;
            if (t < L) s0 = s;
            sum += s;
        }
        float up = a.sigmoid ? a.scale : a.scale / zsum;
        if (a.renormalize) up = a.scale / (lanes_addf<L>(sum) + expf(log_eps - m));
        for (int t = p; t < k; t += L) {
            if (!real) break;
            const int e = t < L ? e0 : t < found ? s_idx[t] : -1;
            const float s = t < L ? s0 : e >= 0 ? score(Elt<T>::to_f32(l[e])) : 0.0f;
            a.idx[row * k + t] = e;
            a.w[row * k + t] = e >= 0 ? up * s : 0.0f;
            if (hist && e >= 0) atomicAdd(&s_hist[e], 1);
        }
        wave_sync();
    }
    if (!hist) return;
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) a.counts[e] = s_hist[e];
}

// Lanes and values: the fewest lanes that hold a row with at most 16 values each, each
// group on lanes of its own; more lanes where the call has too few rows to give every
// SIMD a wave (4,744 rows of 64 bf16: 8 lanes, 593 waves, 11.5 us; 16, 1,186 waves, 4.9;
// 64, 4,744 waves, 7.2).  32,768 rows of 256: 16 lanes 21.8 us, 32 lanes 29, 64 lanes 48 (what
// a row costs beyond its keys is then paid for fewer rows at once).
RouteShape route_shape(int64_t rows, int E, int groups) {
    RouteShape s{};
    int gp = 1;
    while (gp < groups) gp <<= 1;
    s.per = E / groups;
    for (s.L = std::max(8, gp);; s.L <<= 1) {
        s.lanes = s.L / gp;
        s.each = (s.per + s.lanes - 1) / s.lanes;
        if (s.L == kWave || (s.each <= 16 && (s.each == 1 || rows * s.L / kWave >= kRouteWavesMin))) break;
    }
    for (s.V = 1; s.V < s.each; s.V <<= 1) {}
    return s;
}


// ---- the gradient -----------------------------------------------------------------
//
//   S = sum of the chosen s + eps, A = sum of dw s over the chosen (an empty slot, or a masked
//   expert's, has no part in them: its dw is not used)
//   ds_i = scale (dw_i - A / S) / S (renormalised) or scale dw_i, 0 where not chosen
//   sigmoid: dl_i = ds_i s_i (1 - s_i)
//   softmax: dl_e = s_e (ds_e - B), B = sum s ds: of renormalised weights scale A eps / S^2
//
// dw_i - A / S and ds_i - B cancel: a row's only survivor keeps eps' share of dw_i, equal dw no
// more.  So the kernel sums differences.  With eps (a softmax's: eps R / (1 + eps), R the
// scores of the experts not chosen, summed as such) as one more slot of dw 0, A / M is the
// slots' mean, M = sum s + that; from c, the dw of the largest of them,
//   dw_i - A / M = (dw_i - c) + (c eps' - sum s (dw - c)) / M
// and with N = S (softmax: in units in which the row's scores sum to Z, S Z)
//   sigmoid: dl_i = scale s_i (1 - s_i) (dw_i - A / M) / N, M = N
//   softmax: dl_i = scale s_i (dw_i - A / M) / N (chosen: N = M (1 + eps)),
//            dl_e = -scale s_e eps A / N^2 (not chosen)
// A softmax that is not renormalised is the same with R in the place of eps', M = N = Z and
// dl_e = -scale s_e A / N^2.  Where an expert is named twice its slots count each, but its score
// only once in Z: then eps' = eps Z, M = N, and B (as above) is taken off the sum of its slots.
//
// HBM bound: a softmax reads the row once, a sigmoid its chosen logits; every element of
// dlogits is written once.  The lanes of a row hold 16-byte chunks of it; the chosen
// elements are scattered into the row in LDS, and it is stored from there in whole chunks.
template <typename T, int L, int C, bool kSigmoid>
__global__ __launch_bounds__(kRouteThreads) void route_backward_kernel(RouteBackwardArgs a, int vector) {
    constexpr int W = 16 / (int)sizeof(T), kRows = kWave / L;
    static_assert(C * W <= 32, "a bit for each of a lane's elements");
    extern __shared__ __align__(16) float s_rows[];
    const int E = a.E, k = a.k;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, p = lane % L, sub = lane / L;
    float* s_row = s_rows + (wave * kRows + sub) * (L * C * W);
    unsigned* s_bits = reinterpret_cast<unsigned*>(s_row);  // [L] the chosen of each lane's elements, at first
    const int64_t stride = (int64_t)gridDim.x * kRouteWaves * kRows;
    for (int64_t row0 = ((int64_t)blockIdx.x * kRouteWaves + wave) * kRows; row0 < a.rows; row0 += stride) {
        const int64_t row = min(row0 + sub, a.rows - 1);
        const bool real = row0 + sub < a.rows;
        const T* l = static_cast<const T*>(a.logits) + row * E;
        // a slot's expert (-1: empty, whatever its value is), value and logit
        const int32_t* idx = a.idx + row * k;
        const float* dw = a.dw + row * k;
        auto read = [&](int t, float* d, float* v) {
            const int e = idx[t];
            *d = dw[t];
            *v = e >= 0 && e < E ? Elt<T>::to_f32(l[e]) : -INFINITY;
            if (*v != -INFINITY) return e;
            *d = 0.0f;
            return -1;
        };
        // lane t's first slot is slot t
        int e0 = -1;
        float d0 = 0.0f, v0 = -INFINITY;
        if (p < k) e0 = read(p, &d0, &v0);
        float s[C][W], top = 0.0f, z = 1.0f;
        if constexpr (!kSigmoid) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = (c * L + p) * W;
                if (vector && at < E) {
                    load16(l + at, s[c]);
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) s[c][i] = at + i < E ? Elt<T>::to_f32(l[at + i]) : -INFINITY;
                }
            }
            top = s[0][0];
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < W; ++i) top = fmaxf(top, s[c][i]);
            top = lanes_maxf<L>(top);
            if (top == -INFINITY) top = 0.0f;
            z = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < W; ++i) z += s[c][i] = __builtin_amdgcn_exp2f((s[c][i] - top) * 1.44269504f);
            z = lanes_addf<L>(z);
        }
        // what is chosen, and whether anything is twice
        s_bits[p] = 0;
        wave_sync();
        bool some = false, twice = false;
        float most = -INFINITY;
        for (int t = p; t < k; t += L) {
            int e = e0;
            float d = d0, v = v0;
            if (t >= L) e = read(t, &d, &v);
            if (e < 0) continue;
            const int chunk = e / W;
            const unsigned bit = 1u << (chunk / L * W + e % W);
            twice |= (atomicOr(&s_bits[chunk % L], bit) & bit) != 0;
            some = true;
            most = fmaxf(most, v);
        }
        wave_sync();
        const unsigned chosen = s_bits[p];
        wave_sync();
        some = lanes_max<L>(some);
        twice = lanes_max<L>(twice);
        // Renormalised: scores and eps relative to the larger of the largest chosen one and eps, as
        // the forward's weights (a softmax's scores are exp(v - top - m), a sigmoid's s exp(-m)).
        float m = 0.0f, eps = 0.0f;  // eps: times z for a softmax
        if (a.renormalize) {
            most = lanes_maxf<L>(most);
            const float log_eps = a.log_eps + (kSigmoid ? 0.0f : logf(z));
            m = kSigmoid ? fminf(fmaxf(most, log_eps), 0.0f) : fmaxf(most - top, log_eps);
            eps = expf(log_eps - m);
        }
        // a slot's score, and how that moves with the logit
        auto score = [&](float v, float* slope) {
            if constexpr (!kSigmoid) return *slope = expf(v - top - m);
            const float q = expf(-fabsf(v)), r = 1.0f / (1.0f + q);
            const float u = v < 0.0f ? expf(v - m) * r : r;
            *slope = u * (v < 0.0f ? r : q * r);
            return u;
        };
        float u0 = 0.0f, slope0 = 0.0f;
        if (e0 >= 0) u0 = score(v0, &slope0);
        // of slot t, with its score and slope
        auto slot = [&](int t, float* d, float* u, float* slope) {
            if (t < L) {
                *d = d0;
                *u = u0;
                *slope = slope0;
                return e0;
            }
            float v;
            const int e = read(t, d, &v);
            *u = *slope = 0.0f;
            if (e >= 0) *u = score(v, slope);
            return e;
        };
        float up = 0.0f, base = 0.0f, center = 0.0f, shift = 0.0f, inner = 0.0f;
        if (kSigmoid && !a.renormalize) {
            up = a.scale;
        } else {
            if (!a.renormalize) most = lanes_maxf<L>(most);
            float sum = 0.0f, dot = 0.0f, rest = 0.0f;
            center = -INFINITY;
            for (int t = p; t < k; t += L) {
                float d, u, slope;
                const int e = slot(t, &d, &u, &slope);
                sum += u;
                dot += d * u;
                if (e >= 0 && (t < L ? v0 : Elt<T>::to_f32(l[e])) == most) center = fmaxf(center, d);
            }
            if constexpr (!kSigmoid) {
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int i = 0; i < W; ++i) rest += (chosen >> (c * W + i)) & 1 ? 0.0f : s[c][i];
                rest = lanes_addf<L>(rest);
            }
            sum = lanes_addf<L>(sum);
            dot = lanes_addf<L>(dot);
            center = lanes_maxf<L>(center);
            // eps (or the rest) as a slot, and the sum of all
            float other = eps, total = sum + eps;
            if constexpr (!kSigmoid) {
                if (!a.renormalize) {
                    other = rest;
                    total = z;
                } else if (!twice) {
                    other = eps * (rest / z) / (1.0f + a.eps);
                }
            }
            float slope;
            const bool plain = !a.renormalize && twice;  // (its slots' values as they are)
            if (plain || other > score(most, &slope) || !(fabsf(center) < INFINITY)) center = 0.0f;
            float off = 0.0f;
            for (int t = p; t < k; t += L) {
                float d, u;
                if (slot(t, &d, &u, &slope) >= 0) off += u * (d - center);
            }
            off = lanes_addf<L>(off);
            if (some) {
                up = a.scale / total;
                if (!plain) shift = (center * other - off) / (sum + other);
                if constexpr (!kSigmoid) {
                    const float mean = dot / total;
                    base = -up * mean * (a.renormalize ? eps / z : 1.0f);
                    if (twice) inner = a.renormalize ? a.eps * mean : mean;
                }
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                float4 b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if constexpr (!kSigmoid)
                    b = make_float4(base * s[c][i], base * s[c][i + 1], base * s[c][i + 2], base * s[c][i + 3]);
                *reinterpret_cast<float4*>(s_row + (c * L + p) * W + i) = b;
            }
        wave_sync();
        for (int t = p; t < k; t += L) {
            float d, u, slope;
            const int e = slot(t, &d, &u, &slope);
            if (e < 0) continue;
            float ds = (d - center) + shift;
            if (twice) {  // an expert named twice: all its slots' shares, in their order
                ds = -inner;
                for (int o = 0; o < k; ++o)
                    if (idx[o] == e) ds += (dw[o] - center) + shift;
            }
            s_row[e] = slope * (up * ds);
        }
        wave_sync();
        T* out = static_cast<T*>(a.dlogits) + row * E;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (c * L + p) * W;
            float v[W];
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const float4 b = *reinterpret_cast<const float4*>(s_row + at + i);
                v[i] = b.x;
                v[i + 1] = b.y;
                v[i + 2] = b.z;
                v[i + 3] = b.w;
            }
            if (!real || at >= E) continue;
            if (vector) {
                store16(out + at, v);
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (at + i < E) out[at + i] = Elt<T>::from_f32(v[i]);
            }
        }
        wave_sync();
    }
}

template <typename T, int L, int C>
hipError_t launch_route_backward_shape(const RouteBackwardArgs& a, hipStream_t s) {
    constexpr int W = 16 / (int)sizeof(T), rows = kRouteWaves * (kWave / L);
    const int vector = a.E % W == 0 && !(((uintptr_t)a.logits | (uintptr_t)a.dlogits) & 15);
    const int64_t blocks = std::min<int64_t>((a.rows + rows - 1) / rows, kRouteGradBlocks);
    launch_kernel(a.sigmoid ? route_backward_kernel<T, L, C, true> : route_backward_kernel<T, L, C, false>,
                  dim3((unsigned)blocks), dim3(kRouteThreads), rows * L * C * W * 4, s, a, vector);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_route_backward_t(const RouteBackwardArgs& a, hipStream_t s) {
    constexpr int W = 16 / (int)sizeof(T);
    const int chunks = (a.E + W - 1) / W;
    // four chunks a lane where the row has them: more rows of a wave share its work on the
    // slots (32,768 rows of 256 f32: one chunk 15.0 us, two 11.8, four 10.9)
    if (chunks <= 8) return launch_route_backward_shape<T, 8, 1>(a, s);
    if (chunks <= 16) return launch_route_backward_shape<T, 8, 2>(a, s);
    if (chunks <= 32) return launch_route_backward_shape<T, 8, 4>(a, s);
    if (chunks <= 64) return launch_route_backward_shape<T, 16, 4>(a, s);
    if (chunks <= 128) return launch_route_backward_shape<T, 32, 4>(a, s);
    return launch_route_backward_shape<T, 64, 4>(a, s);
}

// ---- the caller's routing -----------------------------------------------------------

// The routing of the caller in the form that the router leaves for the
// dispatch: per row distinct experts in ascending order, then -1; an expert
// outside 0 .. E - 1 is no expert, one named twice has the sum of its weights.
// One block per 64-row chunk, whose histogram it writes.  Every slot is compared
// with its row's others: 2 k^2 LDS reads a row.  5 rows 2.3 us, 4,744 rows top-2 4.3.
__global__ __launch_bounds__(kRouteThreads) void given_kernel(GivenRoutingArgs a) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    const int k = a.k, ks = a.k_slots, n = kRouterRows * k;
    int* s_e = reinterpret_cast<int*>(s_raw);           // [64 k] expert, -1 where none
    float* s_w = reinterpret_cast<float*>(s_e + n);     // [64 k]
    int* s_first = reinterpret_cast<int*>(s_w + n);     // [64 k] expert, -1 where named before too
    int* s_hist = s_first + n;                          // [E_cols]
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
        const int r = i / k * k, e = s_e[i];
        bool first = e >= 0;
        for (int t = r; t < i; ++t) first &= s_e[t] != e;
        s_first[i] = first ? e : -1;
    }
    __syncthreads();
    for (int i = tid; i < nrows * k; i += kRouteThreads) {
        const int r = i / k, e = s_first[i];
        if (e < 0) continue;
        // its place: the experts below it; later mentions add their weights
        int at = 0;
        float w = 0.0f;
        for (int t = r * k; t < r * k + k; ++t) {
            at += s_first[t] >= 0 && s_first[t] < e;
            if (s_e[t] == e) w += s_w[t];
        }
        a.idx[(row0 + r) * ks + at] = e;
        a.w[(row0 + r) * ks + at] = w;
        atomicAdd(&s_hist[e], 1);
    }
    // the empty slots (the dense slot, where there is one, comes last of those taken)
    for (int r = tid; r < nrows; r += kRouteThreads) {
        int live = 0;
        for (int t = 0; t < k; ++t) live += s_first[r * k + t] >= 0;
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

template <typename T, int L, int V>
hipError_t launch_route_shape(const RouteArgs& a, const RouteShape& sh, hipStream_t s) {
    constexpr int rows = kRouteWaves * (kWave / L);
    const int64_t need = (a.rows + rows - 1) / rows;
    const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min(need, kRouteBlocks));
    const uint32_t lds = (uint32_t)(rows * a.k + (blocks == 1 ? a.E : 0)) * 4;
    auto kern = a.bias || a.groups > 1 ? route_kernel<T, L, V, true> : route_kernel<T, L, V, false>;
    launch_kernel(kern, dim3(blocks), dim3(kRouteThreads), lds, s, a, sh);
    if (a.counts && blocks > 1) {
        const int64_t n = a.rows * a.k, most = (n + kCountThreads - 1) / kCountThreads;
        launch_kernel(route_count_kernel, dim3((unsigned)std::min<int64_t>(kCountBlocks, most)), dim3(kCountThreads),
                      0, s, (const int32_t*)a.idx, n, a.E, a.counts);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t launch_route_t(const RouteArgs& a, hipStream_t s) {
    RouteShape sh = route_shape(a.rows, a.E, a.groups);
    const uintptr_t at = (uintptr_t)std::min<size_t>(16, sh.V * sizeof(T)) - 1;
    sh.vector = sh.each == sh.V && sh.per == sh.lanes * sh.V && !((uintptr_t)a.logits & at) &&
                !((a.E * sizeof(T)) & at) && !((uintptr_t)a.bias & (std::min<size_t>(16, sh.V * 4) - 1));
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
    const size_t lds = (size_t)kRouterRows * a.k * 12 + (size_t)a.E_cols * 4;
    constexpr size_t kMost = 160 * 1024;
    if (a.rows < 1 || a.k < 1 || a.k > a.E || lds > kMost) return hipErrorInvalidValue;
    if (lds > 48 * 1024) {
        // (all that there is: calls of several threads set the same value)
        const hipError_t e =
            hipFuncSetAttribute((const void*)given_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kMost);
        if (e != hipSuccess) return e;
    }
    launch_kernel(given_kernel, dim3((unsigned)((a.rows + kRouterRows - 1) / kRouterRows)), dim3(kRouteThreads),
                  (uint32_t)lds, s, a);
    return hipGetLastError();
}

}  // namespace nomas
