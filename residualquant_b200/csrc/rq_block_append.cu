// Append to the 8-bit block-scaled cache: the new tokens' K/V rows are quantized into their blocks.
//
//   amax = largest finite |x| over the block's new tokens          s_need = smallest power of two with amax <= top * s_need
//   s    = s_need for a block that starts here, max(s_old, s_need) for one that held tokens before
//   code = rne(x / s); where s grew, the earlier tokens' codes become rne(code * s_old / s)
//
// One warp owns a (block, KV head, plane) for the whole call: it is the only reader and writer of that scale, so the result
// depends on no order and needs no atomics.  The warp that does the work is the one at the block's first new row (a "leader"
// row: the request's first row, or one whose position starts a block); the tokens stay in registers between the maximum and
// the encoding, so every row is read once.  Memory bound: 2 bytes read and 1 written per element.
#include "rq_block_common.cuh"

namespace rq {
namespace {

constexpr int kAppendWarps = 8;

template <bool INT8>
__device__ __forceinline__ uint2 encode8(const uint4& x, float inverse, bool fp16) {
    const float2 a = activation2(x.x, fp16), b = activation2(x.y, fp16), c = activation2(x.z, fp16), d = activation2(x.w, fp16);
    return make_uint2(encode2<INT8>(a.x * inverse, a.y * inverse) | (encode2<INT8>(b.x * inverse, b.y * inverse) << 16),
                      encode2<INT8>(c.x * inverse, c.y * inverse) | (encode2<INT8>(d.x * inverse, d.y * inverse) << 16));
}

__device__ __forceinline__ uint32_t finite_magnitude(float x) {
    const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
    return bits < 0x7f800000u ? bits : 0u;
}

template <int D, int P, bool INT8>
__global__ void __launch_bounds__(kAppendWarps * 32) block_append_kernel(const BlockAppendParams p) {
    constexpr int kRow = D / 8;             // pieces of eight channels in a row
    constexpr int kPieces = P * kRow / 32;  // pieces a lane holds
    const BlockView& v = p.v;
    const int lane = threadIdx.x & 31;
    const int planes = 2 * v.kv_heads;
    const int64_t warp = static_cast<int64_t>(blockIdx.x) * kAppendWarps + (threadIdx.x >> 5);
    const int64_t piece_of_rows = warp / planes;
    pdl_wait();
    pdl_launch_dependents();
    if (piece_of_rows * p.chunk >= p.num_rows) return;
    const int head = static_cast<int>(warp % planes) >> 1, plane = static_cast<int>(warp % planes) & 1;
    int row = static_cast<int>(piece_of_rows) * p.chunk;
    const int end = min(row + p.chunk, p.num_rows);
    const int64_t page_bytes = static_cast<int64_t>(P) * D;
    const int64_t stride = p.stride[plane];
    const uint16_t* source = static_cast<const uint16_t*>(p.rows[plane]);

    int r = find_request(v.query_start_loc, v.num_requests, row, lane);
    while (row < end && r < v.num_requests) {
        const int first = v.query_start_loc[r], last = min(v.query_start_loc[r + 1], p.num_rows);
        if (row < first) { row = first; continue; }
        if (row >= last) { ++r; continue; }
        const int position = v.seq_lens[r] - (v.query_start_loc[r + 1] - row);
        if (position < 0) { row += min(-position, last - row); continue; }  // rows before the sequence's start hold no token
        const int old = position % P;  // slots of the block that are taken already
        if (old != 0 && row != first) { row += min(P - old, last - row); continue; }
        const int count = min(P - old, last - row);
        const int64_t id = block_id(v, r, position / P);
        if (id >= 0) {
            uint4 x[kPieces];
            uint32_t amax = 0u;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int piece = i * 32 + lane, token = piece / kRow - old, channel = (piece % kRow) * 8;
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (token >= 0 && token < count) {
                    const uint16_t* at = source + (row + token) * stride + head * D + channel;
                    if (p.vector_loads) {
                        x[i] = *reinterpret_cast<const uint4*>(at);
                    } else {
                        x[i] = make_uint4(at[0] | (at[1] << 16), at[2] | (at[3] << 16), at[4] | (at[5] << 16), at[6] | (at[7] << 16));
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint32_t words[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = activation2(words[j], p.fp16);
                    amax = max(amax, max(finite_magnitude(f.x), finite_magnitude(f.y)));
                }
            }
            amax = __reduce_max_sync(kFullMask, amax);
            float* scale_at = v.scales + (static_cast<int64_t>(plane) * v.num_blocks + id) * v.kv_heads + head;
            uint8_t* page = v.codes + ((static_cast<int64_t>(plane) * v.num_blocks + id) * v.kv_heads + head) * page_bytes;
            float before = old != 0 ? *scale_at : 0.f;
            if (!(before > 0.f && before < INFINITY)) before = 0.f;
            float scale = amax != 0u ? block_scale<INT8>(amax) : 0.f;
            scale = fmaxf(scale, before);
            if (scale == 0.f) scale = 1.f;
            if (old != 0 && scale > before) {
                const float ratio = before / scale;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int piece = i * 32 + lane;
                    if (piece / kRow < old) {
                        uint2* at = reinterpret_cast<uint2*>(page + piece * 8);
                        const uint2 c = *at;
                        const float2 a = decode2<INT8>(c.x), b = decode2<INT8>(c.x >> 16), d = decode2<INT8>(c.y), e = decode2<INT8>(c.y >> 16);
                        *at = make_uint2(encode2<INT8>(a.x * ratio, a.y * ratio) | (encode2<INT8>(b.x * ratio, b.y * ratio) << 16),
                                         encode2<INT8>(d.x * ratio, d.y * ratio) | (encode2<INT8>(e.x * ratio, e.y * ratio) << 16));
                    }
                }
            }
            const float inverse = 1.f / scale;  // exact: the scales written here are powers of two
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int piece = i * 32 + lane, token = piece / kRow - old;
                if (token >= 0 && token < count) *reinterpret_cast<uint2*>(page + piece * 8) = encode8<INT8>(x[i], inverse, p.fp16);
            }
            __syncwarp();
            if (lane == 0) *scale_at = scale;
            if (plane == 0 && v.weights != nullptr && lane < count)
                v.weights[(id * v.kv_heads + head) * P + old + lane] = 0.f;
        }
        row += count;
    }
}

template <int D, int P>
cudaError_t launch_append(const BlockAppendParams& p, int int8, cudaStream_t stream) {
    const int64_t warps = (static_cast<int64_t>(p.num_rows) + p.chunk - 1) / p.chunk * 2 * p.v.kv_heads;
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
