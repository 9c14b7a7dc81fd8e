// Attention over the 8-bit block-scaled cache: o = sum_j softmax_j(c q . k_j) v_j with k_j, v_j = block scale * code.
//
// A request's rows times the query heads of a KV head are the queries of one "item": kRows of them, a KV head and the
// request's tokens.  Scores and value sums are tensor-core products with the cached side as the wide operand, so that eight
// queries fill an instruction:
//     S^T [16 tokens x 8 queries]  = K [16 x D] Q^T              (mma m16n8k16, fp16 inputs, fp32 sums)
//     O^T [16 channels x 8 queries] += V^T [16 x 16 tokens] P^T
// Codes become fp16 exactly; a query is brought into fp16's range by a power of two, which costs channels below 2^-28 of its
// largest some of their bits.  Which channel an
// instruction's k index means is free as long as both sides agree, so every thread takes whole 8- or 16-byte pieces of a
// row; V's token pairs are interleaved with byte permutes.  The block scales multiply the scores (K) and go into the
// exponent of the softmax weights (V).
//
// Softmax in one pass, base 2: x = score * log2(e), l = sum 2^(x - m), O = sum 2^(x + log2(v scale) - M + 7) * code with
// references m and M that are raised only when a token exceeds them by 2^8 (any thread of the warp sees one), so most tokens
// need no reduction across threads.  Statistics and sums are fp32.  Separate references for l and O keep blocks of tiny value
// scales from losing either.  A weight that multiplies V is the sum of two fp16 numbers, its upper eleven bits and the rest
// (at most 2^15; off by 2^-22 of itself, or by 2^-31 of the largest one where that is more), with a product for each.  An item
// of up to four queries has both in one instruction: its queries stand in columns 0..3 and again in columns 4..7, where the
// rests are, and the two sums are added up in the end.  (One fp16 number for each weight left sums off by up to 2^-12 of
// their terms' magnitude, which shows where they nearly cancel.  The rests cost 0 to 2 % with up to four queries, 64 sequences x 8192 tokens x 16 heads; 4 % with five
// rows, 92 to 96 us; with sixteen queries, 64 x 8192 x 128/8 heads, 224 became 257 us.)
//
// Memory bound: 2 D bytes for each cached token and KV head.  All items' tokens, in chunks of kChunk and kItemCost chunks
// more for each item, are laid end to end and cut into equal spans, one for each CTA (four per SM, three with sixteen queries;
// all resident), whatever the lengths are; the spans are found on the device from the lengths, so that a captured launch
// stays right.  A span that ends inside an item leaves (m, l, M, O) in the workspace, and a second launch joins those.
// Each warp streams its own 16-token units: one lane has the tensor-memory engine copy a unit's rows of K and V into a ring of
// shared-memory stages.  (Copies by all threads, cp.async, kept the load/store unit busy: 40 sequences x 2200 tokens x 8
// heads took 58 us instead of 46.)  The next item's first units are set off before the warps join the results of this one.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "rq_block_common.cuh"

namespace rq {

__device__ int g_block_attention_status;

struct AttentionLaunch {
    alignas(64) CUtensorMap map;  // the codes as [2 * blocks][heads * page tokens][channels]
    BlockAttentionParams p;
};

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 16;              // tokens of one mma step
constexpr int kChunk = kWarps * kUnit; // tokens that spans are counted in
constexpr int kItemCost = 3;           // chunks' worth of time that a CTA spends on beginning and ending an item
// CTAs on a multiprocessor: registers for four or three (128 or 168 a thread; 128 channels spill 32 to 88 bytes at that).
constexpr int resident(int query_tiles) { return query_tiles == 1 ? 4 : 3; }
constexpr int kJoinWarps = 8;
constexpr uint32_t kWaitLimit = 1u << 22;  // polls of a copy's barrier before the kernel gives up
constexpr float kNever = -1e30f;       // reference of a query that has seen no token
constexpr float kSlack = 8.f;          // a reference is raised when exceeded by this many binades
constexpr float kLift = 7.f;           // softmax weights are held times 2^kLift: at most 2^15 in fp16
constexpr float kLn2 = 0.6931471805599453f;

template <int D_, bool INT8_, int NT_, bool SCORES_>
struct Config {
    static constexpr int D = D_, NT = NT_;
    static constexpr bool kInt8 = INT8_;
    static constexpr bool kScores = SCORES_;          // the scores are left behind, for the accumulated weights
    static constexpr int kRows = 8 * NT;              // queries of an item
    static constexpr int kSteps = D / 16;             // k16 steps of a score, and 16-channel tiles of an output
    static constexpr int kPlane = kUnit * D;          // bytes of one plane of a unit
    static constexpr int kStage = 2 * kPlane;
    // units in flight, the one in use included; its stage is where the warp's sums for eight queries go in the end
    static constexpr int kStages = (D == 64 ? 6 : 3) + (NT == 1 ? 0 : 1);
    static_assert(8 * D * 4 <= kStage, "a warp's sums fit a stage");
    static constexpr int kOffInfo = kWarps * kStages * kStage;        // float4 [warps][stages]: K scale, log2 of V's, tokens
    static constexpr int kOffStat = kOffInfo + kWarps * kStages * 16; // float [warps][8][4]: m, l, M, the stage of the sums
    static constexpr int kOffQuery = kOffStat + kWarps * 8 * 16;      // 16-bit [buffers][rows][D]: a piece's queries
    // sixteen queries would take too many registers: their fp16 fragments stay in shared memory, [n][pair of steps][lane]
    static constexpr bool kSharedQueries = NT > 1;
    // The next piece's queries come in while a slow warp may still take in this one's, unless all warps met in between, as they
    // do over the shared fragments: two buffers, or one.
    static constexpr int kQueryBytes = kRows * D * 2, kQueryBuffers = kSharedQueries ? 1 : 2;
    static constexpr int kOffFragments = kOffQuery + kQueryBuffers * kQueryBytes;
    static constexpr int kOffBarrier = kOffFragments + (kSharedQueries ? kQueryBytes : 0);  // uint64 [warps][stages]
    static constexpr int kOffPlace = kOffBarrier + kWarps * kStages * 8;
    static constexpr int kSmem = kOffPlace + 64;
    static constexpr int kSlot = D + 4;                               // floats a query's partial result takes
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void copy16_or_zero(uint32_t to, const void* from, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void barrier_init(uint32_t barrier) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(barrier) : "memory"); }
__device__ __forceinline__ void barrier_expect(uint32_t barrier, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_done(uint32_t barrier, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(barrier), "r"(parity) : "memory");
    return done != 0;
}
// A copy did not arrive in time (no case is known): the call's results are not to be used.  No copy was set off after that, and
// the limit passes once more, for those that were on their way, before the shared memory is given up.
__device__ __noinline__ void give_up(uint32_t barrier) {
    atomicExch(&g_block_attention_status, RQ_ERR_DEVICE_TIMEOUT);
    for (uint32_t polls = 0; polls < kWaitLimit; ++polls) static_cast<void>(barrier_done(barrier, 0u));
}
// kUnit tokens of a head from one page, rows row .. row + 15 of block `block` of the map.
__device__ __forceinline__ void copy_unit(uint32_t to, const CUtensorMap* map, int row, int block, uint32_t barrier) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(to), "l"(map), "r"(0), "r"(row), "r"(block), "r"(barrier) : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A float's upper eleven bits: exact in fp16 from 2^-14 on.
__device__ __forceinline__ float upper_bits(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// x = from - x, in threads where `here`.
__device__ __forceinline__ void subtract_where(float (&x)[4], const float (&from)[4], bool here) {
    asm("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %8, 0;\n\t@p sub.f32 %0, %4, %0;\n\t@p sub.f32 %1, %5, %1;\n\t@p sub.f32 %2, %6, %2;\n\t@p sub.f32 %3, %7, %3;\n\t}"
        : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]) : "f"(from[0]), "f"(from[1]), "f"(from[2]), "f"(from[3]), "r"(static_cast<int>(here)));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Where 16-byte piece `piece` of token `token` stands in a plane of a stage.  128-byte rows have their pieces rotated by xor
// with the token (the copy's 128-byte swizzle), so that the reads of eight rows (K) and of eight pieces of every second row (V)
// meet no bank twice; 64-byte rows the same by pairs (K's reads meet none, V's two); 96-byte rows are packed, and K's 8-byte
// reads meet none, V's 4-byte ones two.
template <int D>
__device__ __forceinline__ int place(int token, int piece) {
    if constexpr (D == 128) return token * 128 + ((piece ^ (token & 7)) << 4);
    if constexpr (D == 96) return token * 96 + (piece << 4);
    return token * 64 + ((piece ^ ((token >> 1) & 3)) << 4);
}

// The work of request r: queries (rows x group), visible tokens, and its share of the chunk list.
struct Request {
    int first, queries, tokens;  // first row, rows * group, tokens that its last row sees at most
    int before;                  // tokens ahead of its first row (may be negative)
    int tiles, chunks;
    int cost;                    // units of work that an item counts: its chunks and a fixed part, or 1 where items are not cut
};
template <int ROWS>
__device__ __forceinline__ Request request_from(const BlockAttentionParams& p, int first, int last, int length) {
    Request q;
    q.first = first;
    q.queries = max(0, min(last, p.num_rows) - first) * p.group;
    q.tokens = max(0, min(length, p.max_len));
    q.before = length - (last - first);
    q.tiles = (q.queries + ROWS - 1) / ROWS;
    q.chunks = max(1, (q.tokens + kChunk - 1) / kChunk);
    q.cost = p.whole_items ? 1 : q.chunks + kItemCost;
    return q;
}
template <int ROWS>
__device__ __forceinline__ Request request_of(const BlockAttentionParams& p, int r) {
    return request_from<ROWS>(p, p.v.query_start_loc[r], p.v.query_start_loc[r + 1], p.v.seq_lens[r]);
}
__device__ __forceinline__ int64_t work_of(const BlockAttentionParams& p, const Request& q) {
    return static_cast<int64_t>(q.tiles) * p.v.kv_heads * q.cost;
}

// Where things stand in the list of all items: each takes kItemCost units and one for each chunk, and the list is cut into
// spans.  Finds the sum of all requests' units, and the request that span `at` begins in with the units before it.  All
// threads of the block take part.
struct Place {
    int64_t total, before, span;
    int request;
};
template <int WARPS>
struct PlaceShared {
    int64_t warp_sums[WARPS];
    int64_t before;
    int request;
};
template <int ROWS, int WARPS>
__device__ __forceinline__ Place find_place(const BlockAttentionParams& p, PlaceShared<WARPS>& shared, int at) {
    const int n = p.v.num_requests, each = (n + WARPS * 32 - 1) / (WARPS * 32);
    const int lo = min(n, static_cast<int>(threadIdx.x) * each), hi = min(n, lo + each);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t sum = 0;
    for (int r = lo; r < hi; ++r) sum += work_of(p, request_of<ROWS>(p, r));
    int64_t inclusive = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t other = __shfl_up_sync(kFullMask, inclusive, o);
        if (lane >= o) inclusive += other;
    }
    if (lane == 31) shared.warp_sums[warp] = inclusive;
    __syncthreads();
    Place place;
    place.total = 0;
    int64_t running = inclusive - sum;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) running += shared.warp_sums[w];
        place.total += shared.warp_sums[w];
    }
    place.span = max(static_cast<int64_t>(1), (place.total + p.spans - 1) / p.spans);
    const int64_t target = at * place.span;
    if (running <= target && target < running + sum) {
        for (int r = lo; r < hi; ++r) {
            const int64_t one = each == 1 ? sum : work_of(p, request_of<ROWS>(p, r));
            if (target < running + one) {
                shared.before = running;
                shared.request = r;
                break;
            }
            running += one;
        }
    }
    __syncthreads();
    place.before = shared.before;
    place.request = shared.request;
    return place;
}

// A query's row in its request and its head in the group (mostly there is one row, and no division).
struct RowHead {
    int row, head;
};
__device__ __forceinline__ RowHead row_and_head(int query, int group) {
    if (query < group) return {0, query};
    const int row = query / group;
    return {row, query - row * group};
}

// Writes one query's finished output channels (four of them) and, from one thread of it, its lse.
__device__ __forceinline__ void write_output(const BlockAttentionParams& p, int row, int head, int D, int channel, float4 o, float m,
                                             float l, float M) {
    const float factor = l == 0.f ? 0.f : exp2_fast(M - kLift - m) / l;
    uint16_t* to = static_cast<uint16_t*>(p.output) + row * p.output_stride + head * D + channel;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_activation2(o.x * factor, o.y * factor, p.fp16),
                                               pack_activation2(o.z * factor, o.w * factor, p.fp16));
    if (channel == 0) {
        const float lse = l == 0.f ? -INFINITY : m + log2_fast(l);
        const int64_t at = static_cast<int64_t>(row) * p.heads + head;
        if (p.lse != nullptr) p.lse[at] = lse * kLn2;
        if (p.row_lse != nullptr) p.row_lse[at] = lse;
    }
}

template <typename C>
__global__ void __launch_bounds__(kThreads, resident(C::NT)) block_attention_kernel(const __grid_constant__ AttentionLaunch launch) {
    const BlockAttentionParams& p = launch.p;
    constexpr int D = C::D, NT = C::NT, kRows = C::kRows, kSteps = C::kSteps, kStages = C::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    static_assert(sizeof(PlaceShared<kWarps>) <= 64, "room for the place");
    PlaceShared<kWarps>& place_shared = *reinterpret_cast<PlaceShared<kWarps>*>(smem + C::kOffPlace);
    const BlockView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int page_shift = v.page_tokens == 16 ? 4 : 5;
    pdl_wait();
    pdl_launch_dependents();
    const Place start = find_place<kRows, kWarps>(p, place_shared, blockIdx.x);
    const int64_t begin = blockIdx.x * start.span, end = min(begin + start.span, start.total);
    if (tid == 0 && !p.whole_items) p.cuts[blockIdx.x].pieces = 0;  // until an item is found that goes on in the next span
    if (begin >= end) return;
    const int64_t plane_scales = v.num_blocks * v.kv_heads;
    uint8_t* ring = smem + warp * kStages * C::kStage;
    const uint32_t ring_address = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    float4* info = reinterpret_cast<float4*>(smem + C::kOffInfo) + warp * kStages;
    float* stats = reinterpret_cast<float*>(smem + C::kOffStat);
    const uint32_t barriers = static_cast<uint32_t>(__cvta_generic_to_shared(smem + C::kOffBarrier)) + warp * kStages * 8;
    if (lane < kStages) barrier_init(barriers + lane * 8);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the barriers are there for the copies
    __syncwarp();
    uint32_t phases = 0u;  // bit s: parity of the copy into stage s that is waited for next
    bool failed = false;   // a copy has not arrived in time

    // The span's pieces, one after the other; all of this but `units` is the same in every thread of the block.
    int64_t at = begin;
    int r = start.request;
    int64_t ahead = start.before;  // units of work ahead of request r
    Request q = request_of<kRows>(p, r);
    int head, query0, token_begin, token_end;
    int units;           // of the piece, this warp's
    bool whole;          // the piece is all of its item
    int more_spans;      // the piece begins its item: spans behind this one that go on with it
    int64_t slot;        // else: where its result goes
    // Windows: lane i holds the page id of the warp's unit 32 w + i (-1: none, or outside the cache) and its scales, and of
    // the window after it the ids from the window's start on and the scales from its middle on.
    int ids, ids_next;
    float key_scales, value_scales, key_scales_next, value_scales_next;
    auto window = [&](int first) {
        const int unit = first + lane;
        const int id = unit < units ? v.block_table[static_cast<int64_t>(r) * v.table_stride + ((token_begin + (warp + unit * kWarps) * kUnit) >> page_shift)] : -1;
        return id < v.num_blocks ? id : -1;
    };
    auto scale = [&](int id, int plane) { return id >= 0 ? v.scales[plane * plane_scales + static_cast<int64_t>(id) * v.kv_heads + head] : 1.f; };
    auto next_piece = [&]() -> bool {
        while (at < end) {
            const int64_t local = at - ahead;
            if (local >= work_of(p, q)) {  // on to the next request that has work (there is one: at < total)
                ahead += work_of(p, q);
                q = request_of<kRows>(p, ++r);
                continue;
            }
            const int cost = q.cost;
            const int item = static_cast<int>(local / cost), done = static_cast<int>(local - static_cast<int64_t>(item) * cost);
            const int upto = static_cast<int>(min(static_cast<int64_t>(cost), done + (end - at)));
            const int chunk0 = p.whole_items ? 0 : max(0, done - kItemCost), chunk1 = p.whole_items ? q.chunks : upto - kItemCost;
            // a span leaves at most two unfinished pieces: one that goes on at its start, and one that begins inside it
            slot = 2LL * blockIdx.x + (at == begin && done >= kItemCost ? 0 : 1);
            at += upto - done;
            if (chunk1 <= chunk0) continue;  // the span ends before the item's first chunk
            whole = chunk0 == 0 && chunk1 == q.chunks;
            more_spans = chunk0 == 0 && !whole ? static_cast<int>((ahead + static_cast<int64_t>(item + 1) * cost - 1) / start.span) - static_cast<int>(blockIdx.x) : 0;
            head = item % v.kv_heads;
            query0 = item / v.kv_heads * kRows;
            token_begin = chunk0 * kChunk;
            token_end = min(chunk1 * kChunk, q.tokens);
            const int all_units = (token_end - token_begin + kUnit - 1) / kUnit;
            units = all_units > warp ? (all_units - warp + kWarps - 1) / kWarps : 0;
            ids = window(0);
            ids_next = window(32);
            return true;
        }
        return false;
    };
    // Sets the copies of a unit off, and says what the unit is.
    auto produce = [&](int unit, int to) {
        if (unit >= units) return;
        if ((unit & 31) == 0 && unit > 0) {
            ids = ids_next;
            ids_next = window(unit + 32);
            key_scales = key_scales_next;
            value_scales = value_scales_next;
        }
        const int id = __shfl_sync(kFullMask, ids, unit & 31);
        const int token0 = token_begin + (warp + unit * kWarps) * kUnit;
        if (lane == 0 && !failed) {
            const uint32_t barrier = barriers + to * 8;
            barrier_expect(barrier, id >= 0 ? C::kStage : 0);
            if (id >= 0) {
                const int row = (head << page_shift) + (token0 & (v.page_tokens - 1));
                copy_unit(ring_address + to * C::kStage, &launch.map, row, id, barrier);
                copy_unit(ring_address + to * C::kStage + C::kPlane, &launch.map, row, static_cast<int>(v.num_blocks) + id, barrier);
            }
        }
        if ((unit & 31) == 0) {
            if (unit == 0) {
                key_scales = scale(ids, 0);
                value_scales = scale(ids, 1);
            }
        } else if ((unit & 31) == 16) {
            key_scales_next = scale(ids_next, 0);
            value_scales_next = scale(ids_next, 1);
        }
    };
    auto describe = [&](int unit, int to) {
        if (unit >= units) return;
        const int id = __shfl_sync(kFullMask, ids, unit & 31);
        const float k = __shfl_sync(kFullMask, key_scales, unit & 31), log_v = log2_fast(__shfl_sync(kFullMask, value_scales, unit & 31));
        const int count = id >= 0 ? min(kUnit, token_end - (token_begin + (warp + unit * kWarps) * kUnit)) : 0;
        if (lane == 0) info[to] = make_float4(k, log_v, __int_as_float(count), 0.f);
    };
    int stage = 0;       // of the next unit to be used
    // The query that a column of the products stands for (up to four queries stand there twice).
    auto folded = [&]() { return NT == 1 && q.queries - query0 <= 4; };
    auto query_of = [&](int column) { return folded() ? column & 3 : column; };
    uint8_t* queries = smem + C::kOffQuery;  // of the piece that was set off last
    auto set_off = [&]() {
        if constexpr (C::kQueryBuffers == 2) queries = queries == smem + C::kOffQuery ? queries + C::kQueryBytes : smem + C::kOffQuery;
        // the piece's queries, ahead of the queue of cache copies (rows behind the item's last are zeros)
        for (int i = tid; i < kRows * (D / 8); i += kThreads) {
            const int query = query0 + query_of(i / (D / 8));
            const bool real = query < q.queries;
            const RowHead at = row_and_head(real ? query : 0, p.group);
            const int row = q.first + at.row, query_head = head * p.group + at.head;
            copy16_or_zero(static_cast<uint32_t>(__cvta_generic_to_shared(queries + i * 16)),
                           static_cast<const uint16_t*>(p.query) + row * p.query_stride + query_head * D + i % (D / 8) * 8, real);
        }
        commit_copies();
        // the piece's first units, into the ring but for the stage that is free
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) produce(i, stage + i < kStages ? stage + i : stage + i - kStages);
    };
    bool more = next_piece();
    if (more) {
        set_off();
        wait_copies();
        __syncthreads();
    }

    while (more) {
        // the queries as fp16
        uint32_t qf[C::kSharedQueries ? 1 : NT][kSteps][2];
        uint4* const fragments = reinterpret_cast<uint4*>(smem + C::kOffFragments) + lane;
        float factor[NT][2];   // score units of queries 8 n + 2 t + {0, 1}
        int limit[NT][2];      // tokens that they see
        int least = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // query 8 n + g, the channels that this thread's K words hold: four of step s, inside its D / 4 contiguous ones
            uint32_t raw[kSteps][2];
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int channel = t * (D / 4) + s * 4;
                const uint2 two = *reinterpret_cast<const uint2*>(queries + ((n * 8 + g) * D + channel) * 2);
                raw[s][0] = two.x;
                raw[s][1] = two.y;
            }
            // the largest magnitude, on the 16-bit patterns; infinities and NaN, if any, are left out one by one
            uint32_t pairs = 0u;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) pairs = __vmaxu2(__vmaxu2(pairs, raw[s][0] & 0x7fff7fffu), raw[s][1] & 0x7fff7fffu);
            uint32_t bits = max(pairs & 0xffffu, pairs >> 16);
            const uint32_t infinity = p.fp16 ? 0x7c00u : 0x7f80u;
            if (bits >= infinity) {
                bits = 0u;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) bits = max(bits, max(finite_or_zero(raw[s][0], infinity), finite_or_zero(raw[s][1], infinity)));
            }
            uint32_t amax = __float_as_uint(activation2(bits, p.fp16).x);
            amax = max(amax, __shfl_xor_sync(kFullMask, amax, 1));
            amax = max(amax, __shfl_xor_sync(kFullMask, amax, 2));
            // The largest magnitude goes to [2^14, 2^15).  bf16 channels down to 2^-31 of it and fp16 ones down to 2^-28 stay
            // exact; smaller ones are off by at most 2^-25, half a step of fp16 there, or 2^-39 of the largest.
            const int e = amax == 0u ? 0 : max(static_cast<int>(amax >> 23) - 127 - 14, -120);
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 f = activation2(raw[s][i], p.fp16);
                    qf[C::kSharedQueries ? 0 : n][s][i] = pack_activation2(f.x * down, f.y * down, true);
                }
            }
            if constexpr (C::kSharedQueries) {  // every warp has all of them, and writes its share
#pragma unroll
                for (int s = 0; s < kSteps; s += 2)
                    if ((n * kSteps + s) / 2 % kWarps == warp) fragments[(n * kSteps + s) / 2 * 32] = make_uint4(qf[0][s][0], qf[0][s][1], qf[0][s + 1][0], qf[0][s + 1][1]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                factor[n][i] = __shfl_sync(kFullMask, up, (2 * t + i) * 4) * p.scale_log2;
                const int column = query0 + query_of(n * 8 + 2 * t + i);
                limit[n][i] = column < q.queries ? max(0, min(q.tokens, q.before + row_and_head(column, p.group).row + 1)) : 0x7fffffff;
                least = min(least, limit[n][i]);
            }
        }
        least = __reduce_min_sync(kFullMask, least);
        const bool fold = folded(), fold_lower = fold && t >= 2;
        if constexpr (C::kSharedQueries) __syncthreads();
        float* score_at[NT][2];
        if constexpr (C::kScores) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int column = query0 + n * 8 + 2 * t + i;
                    const RowHead at = row_and_head(column, p.group);
                    const int64_t query_row = static_cast<int64_t>(q.first + at.row) * p.heads + head * p.group + at.head;
                    score_at[n][i] = column < q.queries ? p.scores + query_row * p.score_stride : nullptr;
                }
            }
        }

        float o[kSteps][NT][4];
        float m[NT][2], M[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[n][i] = M[n][i] = kNever;
                l[n][i] = 0.f;
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) o[s][n][0] = o[s][n][1] = o[s][n][2] = o[s][n][3] = 0.f;
        }

#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) describe(i, stage + i < kStages ? stage + i : stage + i - kStages);
        auto take_units = [&](auto folded_columns) {
            constexpr bool kFold = decltype(folded_columns)::value;
            for (int unit = 0; unit < units; ++unit) {
                const int free_stage = stage == 0 ? kStages - 1 : stage - 1;  // the one that the unit before was in
                __syncwarp();                                                 // no lane reads it any more
                produce(unit + kStages - 1, free_stage);
                describe(unit + kStages - 1, free_stage);
                uint32_t polls = 0;
                while (!barrier_done(barriers + stage * 8, phases >> stage & 1u) && !failed) failed = ++polls > kWaitLimit;
                phases ^= 1u << stage;
                const uint8_t* keys = ring + stage * C::kStage;
                const uint8_t* values = keys + C::kPlane;
                const float4 about = info[stage];
                stage = stage + 1 == kStages ? 0 : stage + 1;
                const int token0 = token_begin + (warp + unit * kWarps) * kUnit;
                const int count = __float_as_int(about.z);

                // scores
                float x[NT][4], x_odd[NT][4];  // two sums, so that half the products wait for one another
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[n][i] = x_odd[n][i] = 0.f;
                }
                uint32_t low[kSteps], high[kSteps];  // K words of tokens g and g + 8
                if constexpr (D == 128) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 a = *reinterpret_cast<const uint4*>(keys + place<D>(g, 2 * t + h));
                        const uint4 b = *reinterpret_cast<const uint4*>(keys + place<D>(g + 8, 2 * t + h));
                        low[4 * h] = a.x; low[4 * h + 1] = a.y; low[4 * h + 2] = a.z; low[4 * h + 3] = a.w;
                        high[4 * h] = b.x; high[4 * h + 1] = b.y; high[4 * h + 2] = b.z; high[4 * h + 3] = b.w;
                    }
                } else if constexpr (D == 64) {
                    const uint4 a = *reinterpret_cast<const uint4*>(keys + place<D>(g, t));
                    const uint4 b = *reinterpret_cast<const uint4*>(keys + place<D>(g + 8, t));
                    low[0] = a.x; low[1] = a.y; low[2] = a.z; low[3] = a.w;
                    high[0] = b.x; high[1] = b.y; high[2] = b.z; high[3] = b.w;
                } else {
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) {
                        if (s & 1) continue;
                        const uint2 a = *reinterpret_cast<const uint2*>(keys + g * 96 + t * 24 + s * 4);
                        const uint2 b = *reinterpret_cast<const uint2*>(keys + (g + 8) * 96 + t * 24 + s * 4);
                        low[s] = a.x; low[s + 1] = a.y;
                        high[s] = b.x; high[s + 1] = b.y;
                    }
                }
#pragma unroll
                for (int s = 0; s < kSteps; s += 2) {
                    uint32_t a[4], b[4];
                    to_half<C::kInt8>(low[s], a[0], a[2]);
                    to_half<C::kInt8>(high[s], a[1], a[3]);
                    to_half<C::kInt8>(low[s + 1], b[0], b[2]);
                    to_half<C::kInt8>(high[s + 1], b[1], b[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if constexpr (C::kSharedQueries) {
                            const uint4 f = fragments[(n * kSteps + s) / 2 * 32];
                            mma(x[n], a, f.x, f.y);
                            mma(x_odd[n], b, f.z, f.w);
                        } else {
                            mma(x[n], a, qf[n][s][0], qf[n][s][1]);
                            mma(x_odd[n], b, qf[n][s + 1][0], qf[n][s + 1][1]);
                        }
                    }
                }
                const float value_scale = about.y;
                const bool masked = count < kUnit || token0 + kUnit > least;
                bool raise = false;
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[n][i] = (x[n][i] + x_odd[n][i]) * (about.x * factor[n][i & 1]);
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int token = g + (i >> 1) * 8;
                            if (token >= count || token0 + token >= limit[n][i & 1]) x[n][i] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        top[n][i] = fmaxf(x[n][i], x[n][i + 2]);
                        raise = raise || top[n][i] > m[n][i] + kSlack || top[n][i] + value_scale > M[n][i] + kSlack;
                    }
                }
                if constexpr (C::kScores) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int token = token0 + g + (i >> 1) * 8;
                            if (score_at[n][i & 1] != nullptr && token < limit[n][i & 1]) score_at[n][i & 1][token] = x[n][i];
                        }
                    }
                }
                if (__any_sync(kFullMask, raise)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float high_x = top[n][i];
#pragma unroll
                            for (int step = 4; step < 32; step <<= 1) high_x = fmaxf(high_x, __shfl_xor_sync(kFullMask, high_x, step));
                            const float m_new = fmaxf(m[n][i], high_x), M_new = fmaxf(M[n][i], high_x + value_scale);
                            const float keep_l = exp2_fast(m[n][i] - m_new), keep_o = exp2_fast(M[n][i] - M_new);
                            m[n][i] = m_new;
                            M[n][i] = M_new;
                            l[n][i] *= keep_l;
#pragma unroll
                            for (int s = 0; s < kSteps; ++s) {
                                o[s][n][i] *= keep_o;
                                o[s][n][i + 2] *= keep_o;
                            }
                        }
                    }
                }
                // weights, as fp16 and the fp16 of what that leaves over; the value scale goes into the exponent
                uint32_t weight[NT][2], rest[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float w[4], upper[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        l[n][i & 1] += exp2_fast(x[n][i] - m[n][i & 1]);
                        w[i] = exp2_fast(x[n][i] + (value_scale + kLift - M[n][i & 1]));
                        upper[i] = upper_bits(w[i]);
                    }
                    if constexpr (kFold) {
                        subtract_where(upper, w, fold_lower);
                    } else {
                        rest[n][0] = transpose8x8(pack_activation2(w[0] - upper[0], w[1] - upper[1], true));
                        rest[n][1] = transpose8x8(pack_activation2(w[2] - upper[2], w[3] - upper[3], true));
                    }
                    weight[n][0] = transpose8x8(pack_activation2(upper[0], upper[1], true));
                    weight[n][1] = transpose8x8(pack_activation2(upper[2], upper[3], true));
                }
                // value sums: tokens 2t, 2t + 1 (a[0], a[1]) and 2t + 8, 2t + 9 (a[2], a[3]); this thread's channels D/8 g ...
                constexpr int kWords = D / 32;
                uint32_t word[4][kWords];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int token = 2 * t + (i & 1) + (i >> 1) * 8;
                    if constexpr (D == 128) {
                        const uint4 a = *reinterpret_cast<const uint4*>(values + place<D>(token, g));
                        word[i][0] = a.x; word[i][1] = a.y; word[i][2] = a.z; word[i][3] = a.w;
                    } else if constexpr (D == 64) {
                        const uint2 a = *reinterpret_cast<const uint2*>(values + place<D>(token, g >> 1) + (g & 1) * 8);
                        word[i][0] = a.x; word[i][1] = a.y;
                    } else {
#pragma unroll
                        for (int w = 0; w < kWords; ++w) word[i][w] = *reinterpret_cast<const uint32_t*>(values + token * 96 + g * 12 + w * 4);
                    }
                }
                if (count < kUnit) {  // whatever stands behind the last token, a weight of 0 must not meet it
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (2 * t + (i & 1) + (i >> 1) * 8 >= count) {
#pragma unroll
                            for (int w = 0; w < kWords; ++w) word[i][w] = 0u;
                        }
                    }
                }
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t a[4];
                        to_half<C::kInt8>(__byte_perm(word[0][w], word[1][w], h == 0 ? 0x5140 : 0x7362), a[0], a[1]);
                        to_half<C::kInt8>(__byte_perm(word[2][w], word[3][w], h == 0 ? 0x5140 : 0x7362), a[2], a[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma(o[2 * w + h][n], a, weight[n][0], weight[n][1]);
                            if constexpr (!kFold) mma(o[2 * w + h][n], a, rest[n][0], rest[n][1]);
                        }
                    }
                }
            }
        };
        if (NT == 1 && fold) take_units(std::true_type{});
        else take_units(std::false_type{});

        // ---- the warps' results are joined, while the next piece's units are on their way ----
        const int done_first = q.first, done_queries = q.queries, done_head = head, done_query0 = query0;
        const bool done_whole = whole, done_fold = fold;
        if (more_spans > 0 && tid == 0) p.cuts[blockIdx.x] = {more_spans + 1, static_cast<int>(slot & 1), q.first, q.queries - query0, query0, head};
        const int64_t done_slot = slot;
        more = next_piece();
        if (more) set_off();
        const int last = stage == 0 ? kStages - 1 : stage - 1;  // the stage that is free
        float* area = reinterpret_cast<float*>(ring + last * C::kStage);
        __syncwarp();  // no lane reads the last unit any more
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int step = 4; step < 32; step <<= 1) l[n][i] += __shfl_xor_sync(kFullMask, l[n][i], step);
                const int column = 2 * t + i;
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                    *reinterpret_cast<float2*>(area + column * D + g * (D / 8) + 2 * s) = make_float2(o[s][n][i], o[s][n][i + 2]);
                if (g == 0)
                    *reinterpret_cast<float4*>(stats + (warp * 8 + column) * 4) = make_float4(m[n][i], l[n][i], M[n][i], __int_as_float(last));
            }
            __syncthreads();
            for (int piece = tid; piece < 8 * (D / 4); piece += kThreads) {
                const int column = piece / (D / 4), channel = piece % (D / 4) * 4;
                const int query = done_query0 + n * 8 + column;
                if (query >= done_queries) continue;
                float4 stat[kWarps];
                float m_all = kNever, M_all = kNever, l_all = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    stat[w] = *reinterpret_cast<const float4*>(stats + (w * 8 + column) * 4);
                    m_all = fmaxf(m_all, stat[w].x);
                    M_all = fmaxf(M_all, stat[w].z);
                }
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const uint8_t* sums = smem + (w * kStages + __float_as_int(stat[w].w)) * C::kStage + (column * D + channel) * 4;
                    float4 part = *reinterpret_cast<const float4*>(sums);
                    if (done_fold) {
                        const float4 lower = *reinterpret_cast<const float4*>(sums + 4 * D * 4);
                        part = make_float4(part.x + lower.x, part.y + lower.y, part.z + lower.z, part.w + lower.w);
                    }
                    const float share = exp2_fast(stat[w].z - M_all);
                    l_all += stat[w].y * exp2_fast(stat[w].x - m_all);
                    sum.x += part.x * share;
                    sum.y += part.y * share;
                    sum.z += part.z * share;
                    sum.w += part.w * share;
                }
                if (done_whole) {
                    const RowHead at = row_and_head(query, p.group);
                    write_output(p, done_first + at.row, done_head * p.group + at.head, D, channel, sum, m_all, l_all, M_all);
                } else {
                    float* to = p.partials + (done_slot * kRows + n * 8 + column) * C::kSlot;
                    *reinterpret_cast<float4*>(to + channel) = sum;
                    if (channel == 0) *reinterpret_cast<float4*>(to + D) = make_float4(m_all, l_all, M_all, 0.f);
                }
            }
            if (n == NT - 1) {
                wait_copies();                                                // the next piece's queries
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // copies into the sums' stages come after the sums
            }
            __syncthreads();  // the sums have been read: their stages are free
        }
    }
    if (failed) give_up(barriers);
}

// Joins the pieces of the items that more than one span took part in.  At most one such item begins in a span; the CTAs of
// row `part` of the grid take every gridDim.y-th of its queries, all of their warps on as few at a time as leave none out.
// kBatch pieces are on their way to a warp at once: many where one item is cut into hundreds, few registers (and all CTAs
// resident: 40 registers for six, 48 bytes spilled) where many are cut in two.
template <typename C, int kBatch>
__global__ void __launch_bounds__(kJoinWarps * 32, kBatch > 2 ? 2 : 6) block_join_kernel(const BlockAttentionParams p) {
    constexpr int D = C::D, kRows = C::kRows, kLanes = D / 4;
    __shared__ float4 sums[kJoinWarps][kLanes];
    __shared__ float4 stats[kJoinWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_launch_dependents();
    const int each = (p.spans + gridDim.x - 1) / gridDim.x, first_span = blockIdx.x * each;  // at most 32
    const bool is_cut = lane < each && first_span + lane < p.spans && p.cuts[first_span + lane].pieces != 0;
    for (uint32_t cuts = __ballot_sync(kFullMask, is_cut); cuts != 0u; cuts &= cuts - 1u) {
        const int span = first_span + __ffs(cuts) - 1;
        const BlockCut cut = p.cuts[span];
        const int queries = min(kRows, cut.queries), parts = gridDim.y;
        int together = 1;  // queries that the CTA works on at a time
        while (together < kJoinWarps && together * parts < queries) together *= 2;
        const int warps = kJoinWarps / together, mine = warp % warps;  // warps that share a query
        for (int base = blockIdx.y * together; base < queries; base += parts * together) {
            const int column = base + warp / warps;
            float m = kNever, M = kNever, l = 0.f;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            if (column < queries) {
                for (int first = mine; first < cut.pieces; first += warps * kBatch) {
                    float4 stat[kBatch], x[kBatch];
    #pragma unroll
                    for (int j = 0; j < kBatch; ++j) {  // (without branches, so that all loads are on their way at once)
                        const int i = min(first + j * warps, cut.pieces - 1);
                        const int64_t slot = 2LL * (span + i) + (i == 0 ? cut.inside : 0);
                        const float* from = p.partials + (slot * kRows + column) * C::kSlot;
                        stat[j] = __ldcg(reinterpret_cast<const float4*>(from + D));
                        x[j] = __ldcg(reinterpret_cast<const float4*>(from + (lane < kLanes ? lane * 4 : 0)));
                    }
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        if (first + j * warps >= cut.pieces) stat[j] = make_float4(kNever, 0.f, kNever, 0.f);
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        const float m_new = fmaxf(m, stat[j].x), M_new = fmaxf(M, stat[j].z);
                        l = l * exp2_fast(m - m_new) + stat[j].y * exp2_fast(stat[j].x - m_new);
                        const float keep = exp2_fast(M - M_new), share = first + j * warps < cut.pieces ? exp2_fast(stat[j].z - M_new) : 0.f;
                        sum.x = sum.x * keep + x[j].x * share;
                        sum.y = sum.y * keep + x[j].y * share;
                        sum.z = sum.z * keep + x[j].z * share;
                        sum.w = sum.w * keep + x[j].w * share;
                        m = m_new;
                        M = M_new;
                    }
                }
            }
            if (warps > 1) {
                if (lane < kLanes) sums[warp][lane] = sum;
                if (lane == 0) stats[warp] = make_float4(m, l, M, 0.f);
                __syncthreads();
                if (mine == 0 && column < queries) {
                    for (int w = 1; w < warps; ++w) {
                        const float4 stat = stats[warp + w], x = sums[warp + w][lane < kLanes ? lane : 0];
                        const float m_new = fmaxf(m, stat.x), M_new = fmaxf(M, stat.z);
                        l = l * exp2_fast(m - m_new) + stat.y * exp2_fast(stat.x - m_new);
                        const float keep = exp2_fast(M - M_new), share = exp2_fast(stat.z - M_new);
                        sum.x = sum.x * keep + x.x * share;
                        sum.y = sum.y * keep + x.y * share;
                        sum.z = sum.z * keep + x.z * share;
                        sum.w = sum.w * keep + x.w * share;
                        m = m_new;
                        M = M_new;
                    }
                }
                __syncthreads();
            }
            if (mine == 0 && column < queries && lane < kLanes) {
                const int query = cut.query0 + column;
                const RowHead at = row_and_head(query, p.group);
                write_output(p, cut.first + at.row, cut.head * p.group + at.head, D, lane * 4, sum, m, l, M);
            }
        }
    }
}

// Adds 2^(score - lse), summed over the rows and query heads of a KV head, to the weights: four tokens a thread.  One thread
// adds to a token's weight in a call, so the sum's order is fixed; the atomic is for requests that share blocks.
__global__ void __launch_bounds__(kThreads) block_weights_kernel(const BlockAttentionParams p) {
    const BlockView& v = p.v;
    const int r = blockIdx.x / v.kv_heads, head = blockIdx.x % v.kv_heads;
    const Request q = request_of<8>(p, r);
    const int page_shift = v.page_tokens == 16 ? 4 : 5;
    int token = (blockIdx.y * kThreads + threadIdx.x) * 4;
    int id = token < q.tokens ? v.block_table[static_cast<int64_t>(r) * v.table_stride + (token >> page_shift)] : -1;
    pdl_wait();
    pdl_launch_dependents();
    while (token < q.tokens) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        // the first row that sees a token stands at the token's position, or is the request's first
        const int first_row = max(0, token - q.before);
        int64_t at = static_cast<int64_t>(q.first + first_row) * p.heads + head * p.group;
        for (int row = first_row; row * p.group < q.queries; ++row, at += p.heads) {
            const int seen = q.before + row + 1 - token;  // of the four
#pragma unroll 4
            for (int h = 0; h < p.group; ++h) {
                const float4 x = *reinterpret_cast<const float4*>(p.scores + (at + h) * p.score_stride + token);
                const float lse = p.row_lse[at + h];
                sum[0] += exp2_fast(x.x - lse);
                if (seen > 1) sum[1] += exp2_fast(x.y - lse);
                if (seen > 2) sum[2] += exp2_fast(x.z - lse);
                if (seen > 3) sum[3] += exp2_fast(x.w - lse);
            }
        }
        if (id >= 0 && id < v.num_blocks) {
            float* to = v.weights + ((static_cast<int64_t>(id) * v.kv_heads + head) << page_shift) + (token & (v.page_tokens - 1));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (token + i < q.tokens && sum[i] != 0.f) atomicAdd(to + i, sum[i]);
        }
        token += gridDim.y * kThreads * 4;
        id = token < q.tokens ? v.block_table[static_cast<int64_t>(r) * v.table_stride + (token >> page_shift)] : -1;
    }
}

// The tensor map of the codes: boxes of kUnit tokens of one head.
cudaError_t describe_codes(const BlockView& v, int head_dim, CUtensorMap* map) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<Encode> known{nullptr};
    Encode encode = known.load(std::memory_order_acquire);
    if (encode == nullptr) {
        void* found = nullptr;
        cudaDriverEntryPointQueryResult status;
        const cudaError_t err = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &found, 12000, cudaEnableDefault, &status);
        if (err != cudaSuccess) return err;
        if (status != cudaDriverEntryPointSuccess || found == nullptr) return cudaErrorNotSupported;
        encode = reinterpret_cast<Encode>(found);
        known.store(encode, std::memory_order_release);
    }
    const cuuint64_t rows = static_cast<cuuint64_t>(v.kv_heads) * v.page_tokens;
    const cuuint64_t sizes[3] = {static_cast<cuuint64_t>(head_dim), rows, 2 * static_cast<cuuint64_t>(v.num_blocks)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_dim), rows * head_dim};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(head_dim), kUnit, 1}, steps[3] = {1, 1, 1};
    const CUtensorMapSwizzle swizzle = head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE;
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, v.codes, sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

template <int D, bool INT8, int NT, bool SCORES>
cudaError_t launch(const BlockAttentionParams& p, cudaStream_t stream) {
    using C = Config<D, INT8, NT, SCORES>;
    static std::atomic<uint64_t> prepared{0};  // devices whose shared-memory limit was raised
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if ((device >= 64 || !(prepared.load(std::memory_order_relaxed) >> device & 1))) {
        err = cudaFuncSetAttribute(block_attention_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (err == cudaSuccess) err = cudaFuncSetAttribute(block_attention_kernel<C>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (err != cudaSuccess) return err;
        if (device < 64) prepared.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    const bool programmatic = p.programmatic_launch != 0;
    AttentionLaunch launch;
    launch.p = p;
    if ((err = describe_codes(p.v, D, &launch.map)) != cudaSuccess) return err;
    err = launch_chained(block_attention_kernel<C>, launch, dim3(static_cast<unsigned>(p.spans)), kThreads, C::kSmem, 1, programmatic, stream);
    if (err == cudaSuccess && !p.whole_items)
        err = launch_chained(p.join_parts > 2 ? block_join_kernel<Config<D, INT8, NT, false>, 8> : block_join_kernel<Config<D, INT8, NT, false>, 2>, p,
                             dim3(static_cast<unsigned>(p.join_ctas), static_cast<unsigned>(p.join_parts)), kJoinWarps * 32, 0, 1, programmatic, stream);
    if (err == cudaSuccess && SCORES) {
        const unsigned parts = static_cast<unsigned>(std::min(64, (p.max_len + 4 * kThreads - 1) / (4 * kThreads)));
        if (parts > 0)
            err = launch_chained(block_weights_kernel, p, dim3(static_cast<unsigned>(p.v.num_requests) * p.v.kv_heads, parts), kThreads, 0, 1,
                                 programmatic, stream);
    }
    return err;
}

template <int D, bool INT8>
cudaError_t launch_tiles(const BlockAttentionParams& p, cudaStream_t stream) {
    if (p.query_tiles == 1) return p.accumulate ? launch<D, INT8, 1, true>(p, stream) : launch<D, INT8, 1, false>(p, stream);
    return p.accumulate ? launch<D, INT8, 2, true>(p, stream) : launch<D, INT8, 2, false>(p, stream);
}

}  // namespace

int block_attention_slot_floats(int head_dim, int query_tiles) { return 8 * query_tiles * (head_dim + 4); }
cudaError_t block_attention_status(cudaStream_t stream, int* status) {
    const cudaError_t err = cudaMemcpyFromSymbolAsync(status, g_block_attention_status, sizeof(*status), 0, cudaMemcpyDeviceToHost, stream);
    return err == cudaSuccess ? cudaStreamSynchronize(stream) : err;
}

int64_t block_attention_units(int tokens) { return (tokens + kChunk - 1) / kChunk + kItemCost; }
int block_attention_resident(int query_tiles) { return resident(query_tiles); }

cudaError_t launch_block_attention(const BlockAttentionParams& p, int head_dim, int int8, cudaStream_t stream) {
    if (head_dim == 128) return int8 ? launch_tiles<128, true>(p, stream) : launch_tiles<128, false>(p, stream);
    if (head_dim == 96) return int8 ? launch_tiles<96, true>(p, stream) : launch_tiles<96, false>(p, stream);
    return int8 ? launch_tiles<64, true>(p, stream) : launch_tiles<64, false>(p, stream);
}

}  // namespace rq
