// Attention over the 8-bit block-scaled cache: o = sum_j softmax_j(c q . k_j) v_j, k_j and v_j = block scale * code.
// One CTA per (row, query head); its warps share out the tokens, every warp with its own running maximum and sum.
#include "rq_block_common.cuh"

namespace rq {
namespace {

constexpr int kAttentionWarps = 4;
constexpr float kNever = -1e30f;

template <int D, bool INT8>
__device__ __forceinline__ void load_channels(const uint8_t* row, int lane, float (&x)[4]) {
    // lane l holds channels 4l .. 4l + 3 (D / 4 lanes take part)
    x[0] = x[1] = x[2] = x[3] = 0.f;
    if (lane * 4 < D) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(row + lane * 4);
        const float2 a = decode2<INT8>(word), b = decode2<INT8>(word >> 16);
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    }
}

__device__ __forceinline__ void load_query(const BlockAttentionParams& p, int row, int head, int D, int lane, float (&q)[4]) {
    q[0] = q[1] = q[2] = q[3] = 0.f;
    if (lane * 4 < D) {
        const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.query) + row * p.query_stride + head * D + lane * 4);
        const float2 a = activation2(raw.x, p.fp16), b = activation2(raw.y, p.fp16);
        q[0] = a.x; q[1] = a.y; q[2] = b.x; q[3] = b.y;
    }
}

__device__ __forceinline__ float dot(const float (&q)[4], const float (&k)[4]) {
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
    return s;
}

// Tokens that the row at `row` of request r sees.
__device__ __forceinline__ int visible(const BlockAttentionParams& p, int r, int row) {
    const int64_t limit = min(static_cast<int64_t>(p.v.max_blocks) * p.v.page_tokens, static_cast<int64_t>(p.max_len));
    return static_cast<int>(max(static_cast<int64_t>(0), min(limit, static_cast<int64_t>(p.v.seq_lens[r]) - (p.v.query_start_loc[r + 1] - row) + 1)));
}

template <int D, bool INT8>
__global__ void __launch_bounds__(kAttentionWarps * 32) block_attention_kernel(const BlockAttentionParams p) {
    __shared__ float sums[kAttentionWarps][D + 2];
    const BlockView& v = p.v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x / p.heads, head = blockIdx.x % p.heads, kv = head / p.group;
    pdl_wait();
    pdl_launch_dependents();
    const int r = find_request(v.query_start_loc, v.num_requests, row, lane);
    if (r >= v.num_requests) return;
    const int n = visible(p, r, row), P = v.page_tokens;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, top = kNever, total = 0.f;
    load_query(p, row, head, D, lane, q);
    for (int t = warp; t < n; t += kAttentionWarps) {
        const int64_t id = block_id(v, r, t / P);
        if (id < 0) continue;
        const int64_t page = id * v.kv_heads + kv, planes = v.num_blocks * v.kv_heads;
        float k[4], x[4];
        load_channels<D, INT8>(v.codes + (page * P + t % P) * D, lane, k);
        const float s = dot(q, k) * v.scales[page] * p.scale_log2;
        const float next = fmaxf(top, s), keep = exp2f(top - next), e = exp2f(s - next);
        load_channels<D, INT8>(v.codes + ((planes + page) * P + t % P) * D, lane, x);
        const float w = e * v.scales[planes + page];
        total = total * keep + e;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * keep + w * x[i];
        top = next;
    }
    if (lane * 4 < D) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][lane * 4 + i] = o[i];
    }
    if (lane == 0) {
        sums[warp][D] = top;
        sums[warp][D + 1] = total;
    }
    __syncthreads();
    if (warp != 0) return;
    float all = kNever, denominator = 0.f;
    for (int w = 0; w < kAttentionWarps; ++w) all = fmaxf(all, sums[w][D]);
    for (int w = 0; w < kAttentionWarps; ++w) denominator += exp2f(sums[w][D] - all) * sums[w][D + 1];
    const bool empty = denominator == 0.f;
    if (lane * 4 < D) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < kAttentionWarps; ++w) {
            const float share = exp2f(sums[w][D] - all);
            for (int i = 0; i < 4; ++i) x[i] += share * sums[w][lane * 4 + i];
        }
        const float inverse = empty ? 0.f : 1.f / denominator;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.output) + row * p.output_stride + head * D + lane * 4) =
            make_uint2(pack_activation2(x[0] * inverse, x[1] * inverse, p.fp16), pack_activation2(x[2] * inverse, x[3] * inverse, p.fp16));
    }
    if (lane == 0) {
        const float lse = empty ? -INFINITY : all + log2f(denominator);
        if (p.lse != nullptr) p.lse[static_cast<int64_t>(row) * p.heads + head] = lse * 0.69314718056f;
        if (p.accumulate) p.row_lse[static_cast<int64_t>(row) * p.heads + head] = lse;
    }
}

// Adds every token's weight: one warp per (request, KV head, token).
template <int D, bool INT8>
__global__ void __launch_bounds__(128) block_weights_kernel(const BlockAttentionParams p) {
    const BlockView& v = p.v;
    const int lane = threadIdx.x & 31, P = v.page_tokens;
    const int r = blockIdx.x / v.kv_heads, kv = blockIdx.x % v.kv_heads;
    pdl_wait();
    pdl_launch_dependents();
    const int first = v.query_start_loc[r], last = min(v.query_start_loc[r + 1], p.num_rows);
    if (first >= last) return;
    const int n = visible(p, r, v.query_start_loc[r + 1] - 1);
    for (int t = blockIdx.y * 4 + (threadIdx.x >> 5); t < n; t += gridDim.y * 4) {
        const int64_t id = block_id(v, r, t / P);
        if (id < 0) continue;
        const int64_t page = id * v.kv_heads + kv;
        float k[4], added = 0.f;
        load_channels<D, INT8>(v.codes + (page * P + t % P) * D, lane, k);
        for (int row = first; row < last; ++row) {
            if (t >= visible(p, r, row)) continue;
            for (int h = kv * p.group; h < (kv + 1) * p.group; ++h) {
                float q[4];
                load_query(p, row, h, D, lane, q);
                added += exp2f(dot(q, k) * v.scales[page] * p.scale_log2 - p.row_lse[static_cast<int64_t>(row) * p.heads + h]);
            }
        }
        if (lane == 0) atomicAdd(v.weights + page * P + t % P, added);
    }
}

template <int D, bool INT8>
cudaError_t launch(const BlockAttentionParams& p, cudaStream_t stream) {
    const bool programmatic = p.programmatic_launch != 0;
    cudaError_t err = launch_chained(block_attention_kernel<D, INT8>, p, dim3(static_cast<unsigned>(p.num_rows) * p.heads),
                                     kAttentionWarps * 32, 0, 1, programmatic, stream);
    if (err == cudaSuccess && p.accumulate)
        err = launch_chained(block_weights_kernel<D, INT8>, p, dim3(static_cast<unsigned>(p.v.num_requests) * p.v.kv_heads, 64), 128, 0, 1,
                             programmatic, stream);
    return err;
}

}  // namespace

cudaError_t launch_block_attention(const BlockAttentionParams& p, int head_dim, int int8, cudaStream_t stream) {
    if (head_dim == 128) return int8 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
    if (head_dim == 96) return int8 ? launch<96, true>(p, stream) : launch<96, false>(p, stream);
    return int8 ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
}

}  // namespace rq
