// Append to the 8-bit block-scaled cache: the new tokens' K/V rows are quantized into their blocks.
//
//   amax = largest finite |x| over the block's new tokens          s_need = smallest power of two with amax <= top * s_need
//   s    = s_need for a block that starts here, max(s_old, s_need) for one that held tokens before
//   code = rne(x / s); where s grew, the earlier tokens' codes become rne(code * s_old / s)
//
// One warp owns a (block, KV head, plane) for the whole call: it is the only reader and writer of that scale, so the result
// depends on no order and needs no atomics.  The warp that does the work is the one at the block's first new row (the
// request's first row, or one whose position starts a block); the tokens stay in registers between the maximum and the
// encoding, so every row is read once.  Finding the request, position and page costs three dependent loads, so a warp goes on
// to other heads and planes of the block where there are warps enough.  Memory bound: 2 bytes read and 1 written per element.
#include <type_traits>

#include "rq_block_common.cuh"

namespace rq {
namespace {

constexpr int kAppendWarps = 8;

// Eight activations -> eight codes, for finite values that the scale, a power of two, brings into range.
template <bool INT8>
__device__ __forceinline__ uint2 encode8_finite(const uint4& x, float inverse, bool fp16) {
    const uint32_t words[4] = {x.x, x.y, x.z, x.w};
    uint32_t pairs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = activation2(words[i], fp16);
        if constexpr (INT8) {
            // x / scale + 1.5 * 2^23 rounds to a whole number (ties to even), whose low byte is the code
            const float magic = 12582912.f;
            pairs[i] = __byte_perm(__float_as_uint(fmaf(f.x, inverse, magic)), __float_as_uint(fmaf(f.y, inverse, magic)), 0x0040);
        } else {
            pairs[i] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * inverse, f.y * inverse), __NV_SATFINITE, __NV_E4M3);
        }
    }
    return make_uint2(__byte_perm(pairs[0], pairs[1], 0x5410), __byte_perm(pairs[2], pairs[3], 0x5410));
}

// The same with infinities and NaN among them, or a scale of any value that the block had before.
template <bool INT8>
__device__ __noinline__ uint2 encode8(uint4 x, float scale, float inverse, bool fp16) {
    const uint32_t words[4] = {x.x, x.y, x.z, x.w};
    uint32_t pairs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = activation2(words[i], fp16);
        pairs[i] = encode2<INT8>(sided_quotient(f.x, scale, inverse), sided_quotient(f.y, scale, inverse));
    }
    return make_uint2(pairs[0] | (pairs[1] << 16), pairs[2] | (pairs[3] << 16));
}

// Largest of two pairs' 16-bit magnitudes, pair by pair.
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b & 0x7fff7fffu); }

// The codes of a block's first `old` tokens under a scale that grew.
template <int D, int P, bool INT8>
__device__ __noinline__ void round_again(uint8_t* page, int old, float ratio) {
    const int lane = threadIdx.x & 31;
    constexpr int kPieces = P * D / 256;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int piece = i * 32 + lane;
        if (piece / (D / 8) < old) {
            uint2* at = reinterpret_cast<uint2*>(page + piece * 8);
            const uint2 c = *at;
            *at = make_uint2(rescale4<INT8>(c.x, ratio), rescale4<INT8>(c.y, ratio));
        }
    }
}

// CTAs on a multiprocessor: the registers that a block's pieces take leave room for four, three or two.
constexpr int append_resident(int block_bytes) { return block_bytes <= 16 * 96 ? 4 : block_bytes <= 16 * 128 ? 3 : 2; }

template <int D, int P, bool INT8>
__global__ void __launch_bounds__(kAppendWarps * 32, append_resident(P * D)) block_append_kernel(const BlockAppendParams p) {
    constexpr int kRow = D / 8;             // pieces of eight channels in a row
    constexpr int kPieces = P * kRow / 32;  // pieces of a block that a lane holds
    const BlockView& v = p.v;
    const int lane = threadIdx.x & 31;
    const int strips = 2 * v.kv_heads, groups = (strips + p.strips - 1) / p.strips;  // a strip: one head of one plane
    const int64_t warp = static_cast<int64_t>(blockIdx.x) * kAppendWarps + (threadIdx.x >> 5);
    const int64_t chunk = warp / groups;
    pdl_wait();
    pdl_launch_dependents();
    if (chunk * p.chunk >= p.num_rows) return;
    const int first_strip = static_cast<int>(warp % groups) * p.strips, last_strip = min(strips, first_strip + p.strips);
    int row = static_cast<int>(chunk) * p.chunk;
    const int end = min(row + p.chunk, p.num_rows);

    int r = find_request(v.query_start_loc, v.num_requests, row, lane);
    while (row < end && r < v.num_requests) {
        const int first = v.query_start_loc[r], last = min(v.query_start_loc[r + 1], p.num_rows);
        if (row < first) { row = first; continue; }
        if (row >= last) { ++r; continue; }
        const int position = v.seq_lens[r] - (v.query_start_loc[r + 1] - row);
        if (position < 0) { row += min(-position, last - row); continue; }  // rows before the sequence's start hold no token
        const int old = position % P;  // slots of the block that are taken already
        if (old != 0 && row != first) { row += min(P - old, last - row); continue; }
        const int count = min(P - old, last - row), block_row = row;
        row += count;
        const int64_t id = block_id(v, r, position / P);
        if (id < 0) continue;
        for (int strip = first_strip; strip < last_strip; ++strip) {
            const int plane = strip >= v.kv_heads ? 1 : 0, head = strip - plane * v.kv_heads;
            const int64_t stride = p.stride[plane];
            const uint16_t* source = static_cast<const uint16_t*>(p.rows[plane]) + block_row * stride + head * D;
            uint4 x[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int piece = i * 32 + lane, token = piece / kRow - old, channel = (piece % kRow) * 8;
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (token >= 0 && token < count) {
                    const uint16_t* at = source + token * stride + channel;
                    if (p.vector_loads) {
                        x[i] = *reinterpret_cast<const uint4*>(at);
                    } else {
                        x[i] = make_uint4(at[0] | (at[1] << 16), at[2] | (at[3] << 16), at[4] | (at[5] << 16), at[6] | (at[7] << 16));
                    }
                }
            }
            const int64_t page_index = (plane * v.num_blocks + id) * v.kv_heads + head;
            float* scale_at = v.scales + page_index;
            uint8_t* page = v.codes + page_index * (P * D);
            float before = old != 0 ? *scale_at : 0.f;
            if (!(before > 0.f && before < INFINITY)) before = 0.f;
            // the largest magnitude, on the 16-bit patterns: they are ordered like the values
            const uint32_t infinity = p.fp16 ? 0x7c00u : 0x7f80u;
            uint32_t largest = 0u;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) largest = larger(larger(larger(larger(largest, x[i].x), x[i].y), x[i].z), x[i].w);
            uint32_t bits = __reduce_max_sync(kFullMask, max(largest & 0xffffu, largest >> 16));
            const bool finite = bits < infinity;
            if (!finite) {
                bits = 0u;
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
                    bits = max(bits, max(max(finite_or_zero(x[i].x, infinity), finite_or_zero(x[i].y, infinity)),
                                         max(finite_or_zero(x[i].z, infinity), finite_or_zero(x[i].w, infinity))));
                bits = __reduce_max_sync(kFullMask, bits);
            }
            const uint32_t amax = __float_as_uint(activation2(bits, p.fp16).x);
            float scale = fmaxf(amax != 0u ? block_scale<INT8>(amax) : 0.f, before);
            if (scale == 0.f) scale = 1.f;
            if (old != 0 && scale > before) {
                round_again<D, P, INT8>(page, old, before / scale);
            }
            // every scale written here is a power of two, but the block may have come with another
            const bool plain = finite && power_of_two(scale);
            const float inverse = 1.f / scale;
            auto write_codes = [&](auto finite_power) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int piece = i * 32 + lane, token = piece / kRow - old;
                    if (token >= 0 && token < count) {
                        if constexpr (decltype(finite_power)::value) *reinterpret_cast<uint2*>(page + piece * 8) = encode8_finite<INT8>(x[i], inverse, p.fp16);
                        else *reinterpret_cast<uint2*>(page + piece * 8) = encode8<INT8>(x[i], scale, inverse, p.fp16);
                    }
                }
            };
            if (plain) write_codes(std::true_type{});
            else write_codes(std::false_type{});
            __syncwarp();  // every lane has read the scale
            if (lane == 0) *scale_at = scale;
            if (plane == 0 && v.weights != nullptr && lane < count) v.weights[(id * v.kv_heads + head) * P + old + lane] = 0.f;
        }
    }
}

template <int D, int P>
cudaError_t launch_append(const BlockAppendParams& p, int int8, cudaStream_t stream) {
    const int64_t warps = (static_cast<int64_t>(p.num_rows) + p.chunk - 1) / p.chunk * ((2 * p.v.kv_heads + p.strips - 1) / p.strips);
    const dim3 grid(static_cast<unsigned>((warps + kAppendWarps - 1) / kAppendWarps));
    const bool programmatic = p.programmatic_launch != 0;
    return int8 ? launch_chained(block_append_kernel<D, P, true>, p, grid, kAppendWarps * 32, 0, 1, programmatic, stream)
                : launch_chained(block_append_kernel<D, P, false>, p, grid, kAppendWarps * 32, 0, 1, programmatic, stream);
}

template <int D>
cudaError_t launch_append_page(const BlockAppendParams& p, int int8, cudaStream_t stream) {
    return p.v.page_tokens == 16 ? launch_append<D, 16>(p, int8, stream) : launch_append<D, 32>(p, int8, stream);
}

}  // namespace

cudaError_t launch_block_append(const BlockAppendParams& p, int head_dim, int int8, cudaStream_t stream) {
    if (head_dim == 128) return launch_append_page<128>(p, int8, stream);
    if (head_dim == 96) return launch_append_page<96>(p, int8, stream);
    return launch_append_page<64>(p, int8, stream);
}

}  // namespace rq
