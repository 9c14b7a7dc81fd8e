// Device helpers of the 8-bit block-scaled cache kernels: element conversions, the scale rule, launch plumbing.
#pragma once

#include "rq_common.cuh"
#include "rq_kernels.h"

namespace rq {

constexpr float kTopE4m3 = 448.f, kTopInt8 = 127.f;

// Smallest power of two s >= 2^-100 with amax <= top * s, from the bits of a finite amax > 0: top = 1.75 * 2^8 for e4m3 and
// 1.984375 * 2^6 for int8, so s has amax's exponent less 8 or 6, one more where amax's mantissa is above top's.  A
// subnormal amax reads as exponent -127 and takes the floor.
template <bool INT8>
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    const int exponent = static_cast<int>(amax_bits >> 23) - 127;
    const bool above = (amax_bits & 0x7fffffu) > (INT8 ? 0x7e0000u : 0x600000u);
    const int e = max(exponent - (INT8 ? 6 : 8) + (above ? 1 : 0), -100);
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ bool power_of_two(float x) { return (__float_as_uint(x) & 0x7fffffu) == 0u; }  // of a normal x

// A product, and a quotient given the divisor's approximate inverse, in a form that rounds to the few bits of a code as the exact
// values would, ties included: a number next to it on the same side of every shorter number, or itself where that is exact.
__device__ __forceinline__ float sided_product(float a, float b) {
    const float p = __fmul_rz(a, b);  // and the last bit set where anything was left over
    return fabsf(fmaf(a, b, -p)) > 0.f ? __uint_as_float(__float_as_uint(p) | 1u) : p;
}
__device__ __forceinline__ float sided_quotient(float a, float b, float inverse) {
    const float q = a * inverse, t = __uint_as_float((__float_as_uint(q) + 0x80u) & 0xffffff00u);  // 16 bits of it
    const float left = fmaf(-t, b, a);                                                            // its sign is exact
    if (!(fabsf(left) > 0.f)) return left == 0.f ? t : q;                                         // infinities and NaN: q
    return __uint_as_float(__float_as_uint(t) + ((left > 0.f) == (__float_as_int(t) >= 0) ? 1u : ~0u));
}

// Two cached bytes -> two floats (exact).
template <bool INT8>
__device__ __forceinline__ float2 decode2(uint32_t pair) {
    if constexpr (INT8) {
        return make_float2(static_cast<float>(static_cast<int8_t>(pair & 0xffu)), static_cast<float>(static_cast<int8_t>((pair >> 8) & 0xffu)));
    } else {
        return __half22float2(fp8x2_to_half2(pair));
    }
}

// Two floats -> two cached bytes: nearest even, infinities saturate, NaN becomes 0.
template <bool INT8>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
    if constexpr (INT8) {
        const int x = max(-127, min(127, __float2int_rn(a))), y = max(-127, min(127, __float2int_rn(b)));  // NaN converts to 0
        return (static_cast<uint32_t>(x) & 0xffu) | ((static_cast<uint32_t>(y) & 0xffu) << 8);
    } else {
        const float2 v = make_float2(a == a ? a : 0.f, b == b ? b : 0.f);
        return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
    }
}

// Four codes times any ratio, rounded to codes again once.
template <bool INT8>
__device__ __forceinline__ uint32_t rescale4(uint32_t word, float ratio) {
    const float2 a = decode2<INT8>(word), b = decode2<INT8>(word >> 16);
    return encode2<INT8>(sided_product(a.x, ratio), sided_product(a.y, ratio)) |
           (encode2<INT8>(sided_product(b.x, ratio), sided_product(b.y, ratio)) << 16);
}

// Four cached bytes -> two fp16 pairs (bytes 0, 1 and bytes 2, 3), exact.  int8: a byte with its sign bit flipped is
// u = code + 128; the fp16 pattern 0x6400 | u is 1024 + u.
template <bool INT8>
__device__ __forceinline__ void to_half(uint32_t word, uint32_t& low, uint32_t& high) {
    if constexpr (INT8) {
        const uint32_t u = word ^ 0x80808080u;
        const __half2 bias = __float2half2_rn(1152.f);
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
        low = *reinterpret_cast<const uint32_t*>(&x);
        high = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(low), "=r"(high) : "r"(word));
    }
}

// A 16-bit activation pair -> two floats.
__device__ __forceinline__ float2 activation2(uint32_t pair, bool fp16) {
    if (fp16) {
        __half2_raw raw;
        raw.x = static_cast<unsigned short>(pair & 0xffffu);
        raw.y = static_cast<unsigned short>(pair >> 16);
        return __half22float2(__half2(raw));
    }
    return make_float2(bf16_bits_to_float(pair & 0xffffu), __uint_as_float(pair & 0xffff0000u));
}

// The larger 16-bit magnitude of a pair, of finite values only.
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t pair, uint32_t infinity) {
    const uint32_t low = pair & 0x7fffu, high = (pair >> 16) & 0x7fffu;
    return max(low < infinity ? low : 0u, high < infinity ? high : 0u);
}

__device__ __forceinline__ uint32_t pack_activation2(float a, float b, bool fp16) {
    if (fp16) {
        const __half2_raw raw = __half2_raw(__floats2half2_rn(a, b));
        return static_cast<uint32_t>(raw.x) | (static_cast<uint32_t>(raw.y) << 16);
    }
    const __nv_bfloat162_raw raw = __nv_bfloat162_raw(__floats2bfloat162_rn(a, b));
    return static_cast<uint32_t>(raw.x) | (static_cast<uint32_t>(raw.y) << 16);
}

// Request that row `row` belongs to: the last r with starts[r] <= row, num_requests for a padding row.  One warp searches
// 32 boundaries at a time; a large batch of single-token requests, where row r is request r, is recognised first.
__device__ __forceinline__ int find_request(const int32_t* starts, int num_requests, int row, int lane) {
    if (num_requests >= 32 && row < num_requests && starts[row] <= row && row < starts[row + 1]) return row;
    int lo = 0, hi = num_requests + 1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step;
        const int count = __popc(__ballot_sync(kFullMask, i < hi && starts[i] <= row));
        if (count == 0) return lo;
        lo += (count - 1) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

__device__ __forceinline__ int64_t block_id(const BlockView& v, int request, int page) {
    if (page >= v.max_blocks) return -1;
    const int id = v.block_table[static_cast<int64_t>(request) * v.table_stride + page];
    return id >= 0 && id < v.num_blocks ? id : -1;
}

template <typename Kernel, typename Params>
cudaError_t launch_chained(Kernel kernel, const Params& p, dim3 grid, int threads, size_t smem, int cluster, bool programmatic,
                           cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    unsigned count = 0;
    if (programmatic) {
        attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[count++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attributes[count].id = cudaLaunchAttributeClusterDimension;
        attributes[count].val.clusterDim.x = cluster;
        attributes[count].val.clusterDim.y = 1;
        attributes[count++].val.clusterDim.z = 1;
    }
    config.attrs = attributes;
    config.numAttrs = count;
    return cudaLaunchKernelEx(&config, kernel, p);
}

}  // namespace rq
