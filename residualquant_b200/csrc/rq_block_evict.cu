// Eviction from the 8-bit block-scaled cache by accumulated attention weight.
//
// Every (request, KV head) is one cluster of CTAs, each with an equal share of the candidates (the tokens that are neither
// among the first `sinks` nor the last `recent`).  Selection: the weights' order-preserving 32-bit keys are read once into shared
// memory; the (budget - sinks - recent) largest are found eleven, eleven and ten bits at a time, by a histogram of the
// candidates that share the digits found so far and the digit at which the count from above reaches what is wanted.  Three
// passes give the key of the last kept candidate and how many candidates equal to it are kept (the first ones); each warp then
// lists the kept tokens of its stretch behind those of the stretches before it.
// Compaction: kept token i moves to position i, and no kept token stands before its new position, so the destination
// blocks are done in ascending waves, a (block, plane) to a warp: a wave reads all its sources into shared memory, the cluster
// meets, then the wave is written.  Later waves read only blocks behind everything written so far, so they can be read ahead.
// Memory bound: weights once, kept tokens once each way.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "rq_block_common.cuh"

namespace rq {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxWarps = 16;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;

// Order-preserving key of a weight: larger weights have larger keys, NaN the lowest, and -0 equals 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t bits = __float_as_uint(w + 0.f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Whether codes times `ratio` are exact in fp16, down to e4m3's and int8's smallest steps: a power of two of moderate size.
__device__ __forceinline__ bool moves_exactly(float ratio) {
    return (__float_as_uint(ratio) & 0x007fffffu) == 0u && ratio >= 6.103515625e-05f && ratio <= 128.f;
}

// Four codes times `ratio`, rounded to codes again; exact products in fp16, one rounding.
template <bool INT8>
__device__ __forceinline__ uint32_t move_codes(uint32_t word, __half2 ratio) {
    uint32_t low, high;
    to_half<INT8>(word, low, high);
    __half2 a = *reinterpret_cast<__half2*>(&low), b = *reinterpret_cast<__half2*>(&high);
    if constexpr (INT8) {
        // + 1536 rounds to a whole number (ties to even), whose low byte is the code
        const __half2 magic = __float2half2_rn(1536.f);
        a = __hfma2(a, ratio, magic);
        b = __hfma2(b, ratio, magic);
        return __byte_perm(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b), 0x6420);
    } else {
        a = __hmul2(a, ratio);
        b = __hmul2(b, ratio);
        return static_cast<uint32_t>(__nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(a), __NV_SATFINITE, __NV_E4M3)) |
               (static_cast<uint32_t>(__nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(b), __NV_SATFINITE, __NV_E4M3)) << 16);
    }
}

// The same for any ratio (not inlined: 32 sequences of 4097 to 9001 tokens take 142 us, inlined 145).
template <bool INT8>
__device__ __noinline__ uint32_t move_codes_any(uint32_t word, float ratio) {
    return rescale4<INT8>(word, ratio);
}

struct EvictShared {
    alignas(16) uint32_t histogram[kBins];          // read in pieces of 16 bytes
    uint32_t greater[kMaxWarps], equal[kMaxWarps];  // a warp's candidates above / at the threshold
    uint32_t digit, above;                          // digit found by a pass, candidates above it
    uint32_t slice;                                 // candidates of all CTAs in this CTA's slice of the bins
    uint32_t all_greater, all_equal;                // this CTA's
};

template <int D, int P, bool INT8>
__global__ void __launch_bounds__(kMaxWarps * 32, P == 16 ? 2 : 1) block_evict_kernel(const BlockEvictParams p) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ EvictShared shared;
    const cg::cluster_group cluster = cg::this_cluster();
    const BlockView& v = p.v;
    const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
    const int pair = blockIdx.x / size;
    const int r = pair / v.kv_heads, head = pair % v.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    auto meet = [&]() {
        if (size == 1) __syncthreads();
        else cluster.sync();
    };
    pdl_wait();
    pdl_launch_dependents();
    const int length = max(0, v.seq_lens[r]);
    const int n = static_cast<int>(min(static_cast<int64_t>(length), static_cast<int64_t>(v.max_blocks) * P));
    const int32_t* table = v.block_table + static_cast<int64_t>(r) * v.table_stride;
    int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.budget;
    if (p.new_lens != nullptr && head == 0 && rank == 0 && tid == 0) p.new_lens[r] = min(length, p.budget);
    if (n <= p.budget) {
        for (int i = rank * threads + tid; i < p.budget; i += size * threads) kept[i] = i < n ? i : -1;
        return;
    }
    auto valid = [&](int id) { return id >= 0 && id < v.num_blocks; };

    // ---- selection ----
    const int candidates = n - p.sinks - p.recent, wanted = p.budget - p.sinks - p.recent;
    const int share = (candidates + size - 1) / size;
    const int from = p.sinks + min(rank * share, candidates), to = p.sinks + min((rank + 1) * share, candidates);
    const int base = from & ~3;                     // keys[i] belongs to token base + i
    const int cached = min(to, base + p.key_room);  // tokens from here on are read again by every pass
    auto key_of = [&](int token) -> uint32_t {
        if (token < cached) return keys[token - base];
        const int id = table[token / P];
        return valid(id) ? weight_key(v.weights[(static_cast<int64_t>(id) * v.kv_heads + head) * P + token % P]) : 0u;
    };
    uint32_t prefix = 0u;
    uint32_t missing = wanted;  // candidates still to be found at or below the prefix
    if (wanted > 0) {
        // four tokens a thread and load, four loads in flight
        for (int token = base + tid * 4; token < cached; token += threads * 16) {
            int id[4];
            float4 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = token + j * threads * 4;
                id[j] = at < cached ? table[at / P] : -1;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = token + j * threads * 4;
                const float nothing = __uint_as_float(0x7fc00000u);
                w[j] = valid(id[j]) ? *reinterpret_cast<const float4*>(v.weights + (static_cast<int64_t>(id[j]) * v.kv_heads + head) * P + at % P)
                                    : make_float4(nothing, nothing, nothing, nothing);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = token + j * threads * 4;
                if (at < cached)
                    *reinterpret_cast<uint4*>(keys + (at - base)) = make_uint4(weight_key(w[j].x), weight_key(w[j].y), weight_key(w[j].z), weight_key(w[j].w));
            }
        }
        constexpr int kShift[4] = {32, 21, 10, 0};
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = kShift[pass + 1], bins = 1 << (kShift[pass] - shift);
            for (int i = tid; i < bins; i += threads) shared.histogram[i] = 0u;
            __syncthreads();
            for (int token = from + tid; token < to; token += threads) {
                const uint32_t key = key_of(token);
                if (pass == 0 || (key >> (kShift[pass] & 31)) == prefix) atomicAdd(&shared.histogram[(key >> shift) & (bins - 1)], 1u);
            }
            // Bins from the top down: the digit is where the count reaches `missing`.  Each CTA of a cluster adds up a slice of all
            // CTAs' bins (slice 0 the topmost), and the one whose slice the count is reached in finds the digit.
            const int width = bins / size, mine_from = bins - (rank + 1) * width;
            meet();
            uint32_t mine[8], sum = 0u;
            const int high = mine_from + width - 1 - tid * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) mine[j] = 0u;
            if (size == 1) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (high - j >= mine_from) mine[j] = shared.histogram[high - j];
            } else if (high >= mine_from) {
#pragma unroll
                for (int c = 0; c < kMaxCluster; ++c) {
                    if (c < size) {
                        const uint4* other = reinterpret_cast<const uint4*>(cluster.map_shared_rank(shared.histogram, (rank + c) % size) + high - 7);
                        const uint4 a = other[0], b = other[1];
                        mine[7] += a.x; mine[6] += a.y; mine[5] += a.z; mine[4] += a.w;
                        mine[3] += b.x; mine[2] += b.y; mine[1] += b.z; mine[0] += b.w;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += mine[j];
            uint32_t inclusive = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t other = __shfl_up_sync(kFullMask, inclusive, o);
                if (lane >= o) inclusive += other;
            }
            if (lane == 31) shared.greater[warp] = inclusive;
            __syncthreads();
            uint32_t running = inclusive - sum;
            for (int w = 0; w < warp; ++w) running += shared.greater[w];
            int owner = 0;
            uint32_t ahead = 0u;  // candidates in the slices above the owner's
            if (size > 1) {
                if (tid == threads - 1) shared.slice = running + sum;
                cluster.sync();
                const uint32_t slice = lane < size ? *cluster.map_shared_rank(&shared.slice, lane % size) : 0u;
                uint32_t upto = slice;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t other = __shfl_up_sync(kFullMask, upto, o);
                    if (lane >= o) upto += other;
                }
                owner = __ffs(__ballot_sync(kFullMask, upto >= missing)) - 1;
                ahead = __shfl_sync(kFullMask, upto - slice, owner);
            }
            if (rank == owner) {
                running += ahead;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (running < missing && running + mine[j] >= missing) {
                        shared.digit = high - j;
                        shared.above = running;
                    }
                    running += mine[j];
                }
            }
            meet();  // the digit is known, and every CTA has read the histograms
            const uint32_t digit = *cluster.map_shared_rank(&shared.digit, owner), above = *cluster.map_shared_rank(&shared.above, owner);
            prefix = (prefix << (kShift[pass] - shift)) | digit;
            missing -= above;
        }
        // candidates above the threshold are kept, and the first `missing` equal to it; a warp takes a contiguous stretch
        const int stretch = ((to - from + warps - 1) / warps + 31) & ~31;
        const int begin = min(to, from + warp * stretch), end = min(to, begin + stretch);
        uint32_t greater = 0u, equal = 0u;
        for (int token = begin + lane; token < end; token += 32) {
            const uint32_t key = key_of(token);
            greater += key > prefix;
            equal += key == prefix;
        }
        greater = __reduce_add_sync(kFullMask, greater);
        equal = __reduce_add_sync(kFullMask, equal);
        if (lane == 0) {
            shared.greater[warp] = greater;
            shared.equal[warp] = equal;
        }
        __syncthreads();
        greater = __reduce_add_sync(kFullMask, lane < warp ? shared.greater[lane] : 0u);  // of the warps before this one
        equal = __reduce_add_sync(kFullMask, lane < warp ? shared.equal[lane] : 0u);
        if (size > 1) {
            if (warp == warps - 1 && lane == 0) {
                shared.all_greater = greater + shared.greater[warp];
                shared.all_equal = equal + shared.equal[warp];
            }
            cluster.sync();
            greater += __reduce_add_sync(kFullMask, lane < rank ? *cluster.map_shared_rank(&shared.all_greater, lane % size) : 0u);
            equal += __reduce_add_sync(kFullMask, lane < rank ? *cluster.map_shared_rank(&shared.all_equal, lane % size) : 0u);
        }
        for (int token0 = begin; token0 < end; token0 += 32) {
            const int token = token0 + lane;
            const uint32_t key = token < end ? key_of(token) : 0u;
            const bool is_greater = token < end && key > prefix, is_equal = token < end && key == prefix;
            const uint32_t above = __ballot_sync(kFullMask, is_greater), at = __ballot_sync(kFullMask, is_equal);
            const uint32_t lower = (1u << lane) - 1u;
            const uint32_t g = greater + __popc(above & lower), e = equal + __popc(at & lower);
            if (is_greater || (is_equal && e < missing)) kept[p.sinks + g + min(e, missing)] = token;
            greater += __popc(above);
            equal += __popc(at);
        }
    }
    for (int i = rank * threads + tid; i < p.sinks + p.recent; i += size * threads) {
        if (i < p.sinks) kept[i] = i;
        else kept[p.budget - p.recent + i - p.sinks] = n - p.recent + i - p.sinks;
    }
    meet();  // the list is complete and visible to the cluster; the keys and other CTAs' shared memory are done with

    // ---- compaction ----
    // A warp's item of a wave goes through three steps, each a wave ahead of the next: where its tokens are (lane i: token i),
    // their codes into shared memory, and the move.
    constexpr int kRow = D / 16;               // 16-byte pieces of a token
    constexpr int kPieces = P * kRow / 32;     // pieces of a block that a lane moves
    uint4* staged = reinterpret_cast<uint4*>(keys) + warp * 2 * P * kRow;
    const int items = 2 * ((p.budget + P - 1) / P), wave = size * warps;
    struct Place {
        int count;            // kept tokens of the block
        int id, slot;         // lane i: page that token i comes from (-1: none) and its slot there
        int to;               // page that the block goes to
        float scale, moved;   // lane i: scale and weight of token i
    };
    auto count_of = [&](int item) { return item < items ? min(P, p.budget - (item >> 1) * P) : 0; };
    auto token_of = [&](int item) { return lane < count_of(item) ? __ldcg(kept + (item >> 1) * P + lane) : 0; };
    auto find = [&](Place& at, int item, int token) {
        at.count = count_of(item);
        at.id = lane < at.count ? table[token / P] : -1;
        at.slot = token % P;
        at.to = at.count > 0 ? table[item >> 1] : -1;
    };
    auto load_scales = [&](Place& at, int item) {
        if (!valid(at.id)) at.id = -1;
        at.scale = at.moved = 0.f;
        if (at.id >= 0) {
            const int64_t page = static_cast<int64_t>(at.id) * v.kv_heads + head;
            at.scale = __ldcg(v.scales + (item & 1) * v.num_blocks * v.kv_heads + page);
            if ((item & 1) == 0) at.moved = __ldcg(v.weights + page * P + at.slot);
        }
    };
    auto load_codes = [&](const Place& at, int item, int stage) {
        const uint8_t* plane = v.codes + (item & 1) * v.num_blocks * v.kv_heads * P * D;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int piece = i * 32 + lane, token = piece / kRow;
            const int id = __shfl_sync(kFullMask, at.id, token), slot = __shfl_sync(kFullMask, at.slot, token);
            const uint8_t* from = plane + (((id >= 0 ? id : 0) * static_cast<int64_t>(v.kv_heads) + head) * P + slot) * D + (piece % kRow) * 16;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(staged + stage * P * kRow + piece))),
                         "l"(from), "r"(id >= 0 ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int item = rank * warps + warp, stage = 0;
    Place now, then;
    const int first_token = token_of(item), next_token = token_of(item + wave);
    int token = token_of(item + 2 * wave);
    find(now, item, first_token);
    find(then, item + wave, next_token);
    load_scales(now, item);
    load_codes(now, item, 0);
    load_scales(then, item + wave);
    for (int done = 0; done < items; done += wave) {
        Place later;
        load_codes(then, item + wave, stage ^ 1);
        find(later, item + 2 * wave, token);
        token = token_of(item + 3 * wave);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        // The vote has every lane's scale and weight arrive as well, before any warp may write to where they came from.
        const bool odd = __any_sync(kFullMask, now.scale != now.scale || now.moved != now.moved);
        // (relaxed: the sources have arrived, and nothing that was written is handed on)
        if (size > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
        uint32_t amax = 0u;
        const uint4* codes = staged + stage * P * kRow + lane;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint4 code = codes[i * 32];
            const uint32_t words[4] = {code.x, code.y, code.z, code.w};
            __half2 largest = __float2half2_rn(0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t low, high;
                to_half<INT8>(words[j], low, high);
                largest = __hmax2(largest, __hmax2(__habs2(*reinterpret_cast<__half2*>(&low)), __habs2(*reinterpret_cast<__half2*>(&high))));
            }
            const float2 both = __half22float2(largest);
            const uint32_t bits = __float_as_uint(__fmul_ru(fmaxf(both.x, both.y), __shfl_sync(kFullMask, now.scale, (i * 32 + lane) / kRow)));
            if (bits < 0x7f800000u) amax = max(amax, bits);
        }
        amax = __reduce_max_sync(kFullMask, amax);
        const float fresh = amax != 0u ? block_scale<INT8>(amax) : 1.f;
        const float own_ratio = now.scale * (1.f / fresh);
        const bool exact = !odd && __all_sync(kFullMask, lane >= now.count || moves_exactly(own_ratio));
        if (size > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every source of this wave has been read
        else __syncthreads();
        const bool write = valid(now.to);
        const int64_t page = static_cast<int64_t>(now.to) * v.kv_heads + head, plane_page = (item & 1) * v.num_blocks * v.kv_heads + page;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int piece = i * 32 + lane;
            const float ratio = __shfl_sync(kFullMask, own_ratio, piece / kRow);
            const uint4 code = codes[i * 32];
            uint32_t words[4] = {code.x, code.y, code.z, code.w};
            if (exact) {
                const __half2 half_ratio = __float2half2_rn(ratio);
#pragma unroll
                for (int j = 0; j < 4; ++j) words[j] = move_codes<INT8>(words[j], half_ratio);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) words[j] = move_codes_any<INT8>(words[j], ratio);
            }
            if (write && piece / kRow < now.count)
                *reinterpret_cast<uint4*>(v.codes + plane_page * P * D + piece * 16) = make_uint4(words[0], words[1], words[2], words[3]);
        }
        if (write && lane == 0) v.scales[plane_page] = fresh;
        if (write && (item & 1) == 0 && lane < now.count) v.weights[page * P + lane] = now.moved;
        load_scales(later, item + 2 * wave);
        now = then;
        then = later;
        item += wave;
        stage ^= 1;
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int D, int P, bool INT8>
cudaError_t launch_evict(const BlockEvictParams& p, cudaStream_t stream) {
    static std::atomic<uint64_t> prepared{0};  // devices whose shared-memory limit was raised
    const auto kernel = block_evict_kernel<D, P, INT8>;
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if (device >= 64 || !(prepared.load(std::memory_order_relaxed) >> device & 1)) {
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(kBlockEvictKeys * 4, kMaxWarps * 2 * P * D));
        if (err != cudaSuccess) return err;
        if (device < 64) prepared.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    const dim3 grid(static_cast<unsigned>(p.v.num_requests) * p.v.kv_heads * p.cluster);
    const size_t staged = static_cast<size_t>(p.threads / 32) * 2 * P * D;
    return launch_chained(kernel, p, grid, p.threads, std::max(static_cast<size_t>(p.key_room) * 4, staged), p.cluster, p.programmatic_launch != 0, stream);
}

template <int D>
cudaError_t launch_evict_variant(const BlockEvictParams& p, int int8, cudaStream_t stream) {
    if (p.v.page_tokens == 16) return int8 ? launch_evict<D, 16, true>(p, stream) : launch_evict<D, 16, false>(p, stream);
    return int8 ? launch_evict<D, 32, true>(p, stream) : launch_evict<D, 32, false>(p, stream);
}

}  // namespace

cudaError_t launch_block_evict(const BlockEvictParams& p, int head_dim, int int8, cudaStream_t stream) {
    if (head_dim == 128) return launch_evict_variant<128>(p, int8, stream);
    if (head_dim == 96) return launch_evict_variant<96>(p, int8, stream);
    return launch_evict_variant<64>(p, int8, stream);
}

}  // namespace rq
