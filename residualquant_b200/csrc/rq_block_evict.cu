// Eviction from the 8-bit block-scaled cache by accumulated attention weight.
//
// Every (request, KV head) is one cluster of CTAs.  Selection: the (budget - sinks - recent) largest of the candidate
// weights are found by their order-preserving 32-bit keys, eleven, eleven and ten bits at a time: a histogram of the
// candidates that share the digits found so far, then the digit at which the count from above reaches what is wanted.  Three
// passes give the key of the last kept candidate and how many candidates equal to it are kept (the first ones).
// Compaction: kept token i moves to position i, and kept positions never exceed their sources, so the destination
// blocks are done in ascending waves: a wave reads all its sources into registers, the cluster meets, then the wave is written.
// Later waves read only blocks behind everything written so far.  Memory bound: weights once, kept tokens once each way.
#include <cooperative_groups.h>

#include "rq_block_common.cuh"

namespace rq {
namespace {

namespace cg = cooperative_groups;

constexpr int kEvictWarps = 16;
constexpr int kEvictThreads = kEvictWarps * 32;
constexpr int kBins = 2048;

// Order-preserving key of a weight: larger weights have larger keys, NaN the lowest, and -0 equals 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t bits = __float_as_uint(w + 0.f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

struct EvictShared {
    uint32_t histogram[kBins];
    uint32_t warp_sums[kEvictWarps];
    uint32_t warp_equal[kEvictWarps];
    uint32_t digit, above;        // digit found by a pass, candidates above it
    uint32_t greater, equal;      // candidates of this CTA above / at the threshold
};

template <int D, bool INT8>
__global__ void __launch_bounds__(kEvictThreads) block_evict_kernel(const BlockEvictParams p) {
    __shared__ EvictShared shared;
    const cg::cluster_group cluster = cg::this_cluster();
    const BlockView& v = p.v;
    const int P = v.page_tokens;
    const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
    const int pair = blockIdx.x / size;
    const int r = pair / v.kv_heads, head = pair % v.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_launch_dependents();
    const int length = max(0, v.seq_lens[r]);
    const int n = static_cast<int>(min(static_cast<int64_t>(length), static_cast<int64_t>(v.max_blocks) * P));
    int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.budget;
    if (p.new_lens != nullptr && head == 0 && rank == 0 && tid == 0) p.new_lens[r] = min(length, p.budget);
    if (n <= p.budget) {
        for (int i = rank * kEvictThreads + tid; i < p.budget; i += size * kEvictThreads) kept[i] = i < n ? i : -1;
        return;
    }
    auto key_of = [&](int token) -> uint32_t {
        const int64_t id = block_id(v, r, token / P);
        return id < 0 ? 0u : weight_key(v.weights[(id * v.kv_heads + head) * P + token % P]);
    };

    // ---- selection ----
    const int candidates = n - p.sinks - p.recent, wanted = p.budget - p.sinks - p.recent;
    const int share = (candidates + size - 1) / size;
    const int from = p.sinks + min(rank * share, candidates), to = p.sinks + min((rank + 1) * share, candidates);
    uint32_t prefix = 0u;
    uint32_t missing = wanted;  // candidates still to be found at or below the prefix
    constexpr int kShift[4] = {32, 21, 10, 0};
    if (wanted > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = kShift[pass + 1], bins = 1 << (kShift[pass] - shift);
            for (int i = tid; i < bins; i += kEvictThreads) shared.histogram[i] = 0u;
            __syncthreads();
            for (int token = from + tid; token < to; token += kEvictThreads) {
                const uint32_t key = key_of(token);
                if (pass == 0 || (key >> kShift[pass]) == prefix) atomicAdd(&shared.histogram[(key >> shift) & (bins - 1)], 1u);
            }
            cluster.sync();
            // bins from the top down, four a thread: the digit is where the running count reaches `missing`
            uint32_t mine[4], sum = 0u;
            const int high = bins - 1 - tid * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mine[j] = 0u;
                if (high - j >= 0)
                    for (int c = 0; c < size; ++c) mine[j] += cluster.map_shared_rank(shared.histogram, c)[high - j];
                sum += mine[j];
            }
            uint32_t inclusive = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t other = __shfl_up_sync(kFullMask, inclusive, o);
                if (lane >= o) inclusive += other;
            }
            if (lane == 31) shared.warp_sums[warp] = inclusive;
            __syncthreads();
            uint32_t running = inclusive - sum;
            for (int w = 0; w < warp; ++w) running += shared.warp_sums[w];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (running < missing && running + mine[j] >= missing) {
                    shared.digit = high - j;
                    shared.above = running;
                }
                running += mine[j];
            }
            cluster.sync();  // the digit is known here, and every CTA has read the histograms
            prefix = (prefix << (kShift[pass] - shift)) | shared.digit;
            missing -= shared.above;
        }
    }
    // candidates above the threshold are kept, and the first `missing` equal to it
    uint32_t greater = 0u, equal = 0u;
    if (wanted > 0) {
        for (int token = from + tid; token < to; token += kEvictThreads) {
            const uint32_t key = key_of(token);
            greater += key > prefix;
            equal += key == prefix;
        }
    }
    greater = __reduce_add_sync(kFullMask, greater);
    equal = __reduce_add_sync(kFullMask, equal);
    if (lane == 0) {
        shared.warp_sums[warp] = greater;
        shared.warp_equal[warp] = equal;
    }
    __syncthreads();
    if (tid == 0) {
        shared.greater = shared.equal = 0u;
        for (int w = 0; w < kEvictWarps; ++w) {
            shared.greater += shared.warp_sums[w];
            shared.equal += shared.warp_equal[w];
        }
    }
    cluster.sync();
    greater = equal = 0u;
    for (int c = 0; c < rank; ++c) {
        greater += *cluster.map_shared_rank(&shared.greater, c);
        equal += *cluster.map_shared_rank(&shared.equal, c);
    }
    if (wanted > 0) {
        for (int base = from; base < to; base += kEvictThreads) {
            const int token = base + tid;
            const uint32_t key = token < to ? key_of(token) : 0u;
            const bool is_greater = token < to && key > prefix, is_equal = token < to && key == prefix;
            const uint32_t above = __ballot_sync(kFullMask, is_greater), at = __ballot_sync(kFullMask, is_equal);
            __syncthreads();
            if (lane == 0) {
                shared.warp_sums[warp] = __popc(above);
                shared.warp_equal[warp] = __popc(at);
            }
            __syncthreads();
            uint32_t g = greater + __popc(above & ((1u << lane) - 1u)), e = equal + __popc(at & ((1u << lane) - 1u));
            for (int w = 0; w < kEvictWarps; ++w) {
                if (w < warp) {
                    g += shared.warp_sums[w];
                    e += shared.warp_equal[w];
                }
                greater += shared.warp_sums[w];
                equal += shared.warp_equal[w];
            }
            if (is_greater || (is_equal && e < missing)) kept[p.sinks + g + min(e, missing)] = token;
        }
    }
    for (int i = rank * kEvictThreads + tid; i < p.sinks + p.recent; i += size * kEvictThreads) {
        if (i < p.sinks) kept[i] = i;
        else kept[p.budget - p.recent + i - p.sinks] = n - p.recent + i - p.sinks;
    }
    cluster.sync();  // the list is complete and visible to the cluster

    // ---- compaction ----
    constexpr int kRow = D / 16;             // 16-byte pieces of a token
    constexpr int kPieces = 32 * kRow / 32;  // pieces a lane holds for a block of 32 tokens
    const int blocks = (p.budget + P - 1) / P;
    const int items = 2 * blocks, wave = size * kEvictWarps;
    for (int base = 0; base < items; base += wave) {
        const int item = base + rank * kEvictWarps + warp;
        const int plane = item & 1, first = (item >> 1) * P;
        const int count = item < items ? min(P, p.budget - first) : 0;
        const int64_t plane_first = static_cast<int64_t>(plane) * v.num_blocks;
        uint4 code[kPieces];
        float scale_of[kPieces];
        float moved = 0.f;
        uint32_t amax = 0u;
        int64_t source = -1;  // page of the lane's token, and its slot and scale
        int slot = 0;
        float scale = 0.f;
        if (lane < count) {
            const int token = __ldcg(kept + first + lane);
            const int64_t id = block_id(v, r, token / P);
            slot = token % P;
            if (id >= 0) {
                source = (plane_first + id) * v.kv_heads + head;
                scale = __ldcg(v.scales + source);
                if (plane == 0) moved = __ldcg(v.weights + (id * v.kv_heads + head) * P + slot);
            }
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int piece = i * 32 + lane, token = piece / kRow;  // token < 32
            const int64_t from_page = __shfl_sync(kFullMask, source, token);
            const int from_slot = __shfl_sync(kFullMask, slot, token);
            scale_of[i] = __shfl_sync(kFullMask, scale, token);
            code[i] = make_uint4(0u, 0u, 0u, 0u);
            if (token < count && from_page >= 0)
                code[i] = __ldcg(reinterpret_cast<const uint4*>(v.codes + (from_page * P + from_slot) * D + (piece % kRow) * 16));
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint32_t words[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 a = decode2<INT8>(words[j]), b = decode2<INT8>(words[j] >> 16);
                const float largest = fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))) * scale_of[i];
                const uint32_t bits = __float_as_uint(largest);
                if (bits < 0x7f800000u) amax = max(amax, bits);
            }
        }
        amax = __reduce_max_sync(kFullMask, amax);
        const float fresh = amax != 0u ? block_scale<INT8>(amax) : 1.f;
        cluster.sync();  // every source of this wave is in registers
        const int64_t id = count > 0 ? block_id(v, r, first / P) : -1;
        if (id >= 0) {
            const int64_t page = (plane_first + id) * v.kv_heads + head;
            const float inverse = 1.f / fresh;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int piece = i * 32 + lane;
                if (piece / kRow >= count) continue;
                uint32_t words[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
                const float ratio = scale_of[i] * inverse;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 a = decode2<INT8>(words[j]), b = decode2<INT8>(words[j] >> 16);
                    words[j] = encode2<INT8>(a.x * ratio, a.y * ratio) | (encode2<INT8>(b.x * ratio, b.y * ratio) << 16);
                }
                *reinterpret_cast<uint4*>(v.codes + page * P * D + static_cast<int64_t>(piece) * 16) =
                    make_uint4(words[0], words[1], words[2], words[3]);
            }
            if (lane == 0) v.scales[page] = fresh;
            if (plane == 0 && lane < count) v.weights[(id * v.kv_heads + head) * P + lane] = moved;
        }
    }
}

template <int D>
cudaError_t launch_evict(const BlockEvictParams& p, int int8, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.v.num_requests) * p.v.kv_heads * p.cluster);
    const bool programmatic = p.programmatic_launch != 0;
    return int8 ? launch_chained(block_evict_kernel<D, true>, p, grid, kEvictThreads, 0, p.cluster, programmatic, stream)
                : launch_chained(block_evict_kernel<D, false>, p, grid, kEvictThreads, 0, p.cluster, programmatic, stream);
}

}  // namespace

cudaError_t launch_block_evict(const BlockEvictParams& p, int head_dim, int int8, cudaStream_t stream) {
    if (head_dim == 128) return launch_evict<128>(p, int8, stream);
    if (head_dim == 96) return launch_evict<96>(p, int8, stream);
    return launch_evict<64>(p, int8, stream);
}

}  // namespace rq
