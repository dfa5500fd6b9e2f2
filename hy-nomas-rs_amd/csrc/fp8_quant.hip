// Values to e4m3 with a scale for each block of 128 (fp8.hpp).
//
// HBM bound: an element is read once and its byte written once; what is between
// them, the quotient rounded exactly, is about 14 instructions an element.  32,768 x 4,096 in bf16 80 us (5.0
// TB/s); squares of 8,192 x 2,048 in f32 18 us a call (4.6 TB/s).  A few thousand rows: a block loads once,
// computes once and stores once, and nothing overlaps these: 4,744 x 2,048 in bf16 10.2 us (2.9 TB/s).
#include "fp8.hpp"

#include <algorithm>

namespace nomas {

namespace {

constexpr int kLanes = 16;  // of a block of 128 columns: 8 columns a lane
constexpr int kQuantThreads = 256;
constexpr int kGroups = kQuantThreads / kLanes;

template <typename T> struct In8 {
    uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ In8<T> fetch(const T* p) {
    In8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void widen(const In8<T>& r, float* o) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) unpack16<T>(r.v[i], o + i * (16 / sizeof(T)));
}
__device__ __forceinline__ uint32_t largest(const float* v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ uint2 pack8(const float* v, const Fp8Quot& d) {
    return make_uint2(fp8_pack4(d(v[0]), d(v[1]), d(v[2]), d(v[3])), fp8_pack4(d(v[4]), d(v[5]), d(v[6]), d(v[7])));
}

// 16 lanes take a block of a row, U blocks a step.
template <typename T, int U>
__global__ __launch_bounds__(kQuantThreads) void quant_rows_kernel(QuantArgs a) {
    const int l = threadIdx.x % kLanes;
    const uint32_t kb = (uint32_t)((a.ld_q + kFp8Block - 1) / kFp8Block), total = (uint32_t)a.rows * kb;
    const T* x = static_cast<const T*>(a.x);
    // (a group's blocks are next to each other for a wave's four groups, U steps apart)
    const uint32_t first = blockIdx.x * (uint32_t)(U * kGroups) + threadIdx.x / kLanes;
    In8<T> in[U];
    uint32_t row[U];
    int col[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const uint32_t u = min(first + i * kGroups, total - 1);
        row[i] = u / kb;
        col[i] = (int)(u - row[i] * kb) * kFp8Block + l * 8;
        in[i] = In8<T>{};
        if (col[i] < a.cols) in[i] = fetch(x + (int64_t)row[i] * a.cols + col[i]);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (first + i * kGroups >= total) break;
        float v[8];
        widen<T>(in[i], v);
        const float s = fp8_scale(max16(largest(v)));
        if (col[i] < a.ld_q) *reinterpret_cast<uint2*>(a.q + (int64_t)row[i] * a.ld_q + col[i]) = pack8(v, Fp8Quot(s));
        if (l == 0) a.scale[(int64_t)row[i] * kb + col[i] / kFp8Block] = s;
    }
}

// A block of threads takes a square, 16 rows at a time; it stays in registers between
// its maximum and its values.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quant_squares_kernel(QuantSquareArgs a) {
    constexpr int P = kFp8Block / kGroups;  // passes over the square's rows
    __shared__ uint32_t s_max[kQuantThreads / kWave];
    const int l = threadIdx.x % kLanes, g = threadIdx.x / kLanes;
    const int rb = blockIdx.y, b = blockIdx.x;
    const int col = b * kFp8Block + l * 8;
    const T* x = static_cast<const T*>(a.x) + blockIdx.z * a.x_batch;
    uint8_t* q = a.q + blockIdx.z * a.q_batch;
    auto at = [&](int i) { return rb * kFp8Block + i * kGroups + g; };  // the logical row
    // ... and where it is stored: groups of 32 rows `row_group` rows apart
    auto stored = [&](int r) { return (int64_t)(r / 32) * a.row_group + r % 32; };
    In8<T> in[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        in[i] = In8<T>{};
        if (at(i) < a.rows && col < a.cols)
            in[i] = fetch(x + (int64_t)(col / 32) * a.x_step + stored(at(i)) * a.x_row + col % 32);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        float v[8];
        widen<T>(in[i], v);
        m = max(m, largest(v));
    }
    m = max16(m);
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    if (threadIdx.x % kWave == 0) s_max[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQuantThreads / kWave; ++w) m = max(m, s_max[w]);
    const float s = fp8_scale(m);
    const Fp8Quot d(s);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        if (at(i) >= a.rows || col >= a.cols) continue;
        float v[8];
        widen<T>(in[i], v);
        const int64_t r = stored(at(i));
        const int64_t to = a.fragments ? ((int64_t)(col / 64) * (a.q_rows / 16) + r / 16) * 1024 + (col / 16 % 4) * 256 +
                                             r % 16 * 16 + col % 16
                                       : r * a.ld_q + col;
        *reinterpret_cast<uint2*>(q + to) = pack8(v, d);
    }
    if (threadIdx.x == 0) a.scale[blockIdx.z * a.scale_batch + (int64_t)rb * gridDim.x + b] = s;
}

}  // namespace

hipError_t launch_quant_rows(DType dt, const QuantArgs& a, hipStream_t s) {
    const int64_t kb = (a.ld_q + kFp8Block - 1) / kFp8Block;
    if (a.rows < 1 || a.cols < 8 || a.cols % 8 != 0 || a.ld_q < a.cols || a.ld_q % 8 != 0 ||
        a.rows * kb >= ((int64_t)1 << 30))  // (four threads a block of 128: 2^32 in a grid)
        return hipErrorInvalidValue;
    constexpr int U = 4;
    const int64_t blocks = (a.rows * kb + U * kGroups - 1) / (U * kGroups);
    const dim3 grid((unsigned)blocks), block(kQuantThreads);
    switch (dt) {
        case DType::F32: launch_kernel(quant_rows_kernel<float, U>, grid, block, 0, s, a); break;
        case DType::BF16: launch_kernel(quant_rows_kernel<__bf16, U>, grid, block, 0, s, a); break;
        case DType::F16: launch_kernel(quant_rows_kernel<_Float16, U>, grid, block, 0, s, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_quant_squares(DType dt, const QuantSquareArgs& a, hipStream_t s) {
    const int64_t kb = (a.cols + kFp8Block - 1) / kFp8Block, rb = (a.rows + kFp8Block - 1) / kFp8Block;
    if (a.rows < 1 || a.cols < 8 || a.cols % 8 != 0 || rb > 65535 || kb > 0x7fffffff || a.batch < 1 || a.batch > 65535)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)kb, (unsigned)rb, (unsigned)a.batch), block(kQuantThreads);
    switch (dt) {
        case DType::F32: launch_kernel(quant_squares_kernel<float>, grid, block, 0, s, a); break;
        case DType::BF16: launch_kernel(quant_squares_kernel<__bf16>, grid, block, 0, s, a); break;
        case DType::F16: launch_kernel(quant_squares_kernel<_Float16>, grid, block, 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace nomas
