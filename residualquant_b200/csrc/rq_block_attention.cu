// Attention over the 8-bit block-scaled cache: o = sum_j softmax_j(c q . k_j) v_j with k_j, v_j = block scale * code.
//
// A request's rows times the query heads of a KV head are the queries of one "item": kRows of them, a KV head and the
// request's tokens.  Scores and value sums are tensor-core products with the cached side as the wide operand, so that eight
// queries fill an instruction:
//     S^T [16 tokens x 8 queries]  = K [16 x D] Q^T              (mma m16n8k16, fp16 inputs, fp32 sums)
//     O^T [16 channels x 8 queries] += V^T [16 x 16 tokens] P^T
// Codes become fp16 exactly, and queries too: each is brought into fp16's range by a power of two.  Which channel an
// instruction's k index means is free as long as both sides agree, so every thread takes whole 8- or 16-byte pieces of a
// row; V's token pairs are interleaved with byte permutes.  The block scales multiply the scores (K) and go into the
// exponent of the softmax weights (V).
//
// Softmax in one pass, base 2: x = score * log2(e), l = sum 2^(x - m), O = sum 2^(x + log2(v scale) - M + 7) * code with
// references m and M that are raised only when a token exceeds them by 2^8 (any thread of the warp sees one), so most tokens
// need no reduction across threads.  Statistics and sums are fp32; the weights that multiply V are fp16 (11 bits, at most
// 2^15, exact to 2^-31 of the largest one below that).  Separate references for l and O keep blocks of tiny value scales
// from losing either.
//
// Memory bound: 2 D bytes for each cached token and KV head.  All items' tokens, in units of kChunk, are laid end to end and
// cut into equal spans, one for each CTA (four per SM, all resident), whatever the lengths are; the spans are found on the
// device from the lengths, so that a captured launch stays right.  A span that ends inside an item leaves (m, l, M, O) in
// the workspace, and a second launch joins those.  Each warp streams its own 16-token units through a ring of cp.async stages.
#include <algorithm>
#include <atomic>

#include "rq_block_common.cuh"

namespace rq {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 16;              // tokens of one mma step
constexpr int kChunk = kWarps * kUnit; // tokens that spans are counted in
constexpr int kStages = 3;
constexpr float kNever = -1e30f;       // reference of a query that has seen no token
constexpr float kSlack = 8.f;          // a reference is raised when exceeded by this many binades
constexpr float kLift = 7.f;           // softmax weights are held times 2^kLift: at most 2^15 in fp16
constexpr float kLn2 = 0.6931471805599453f;

template <int D_, bool INT8_, int NT_>
struct Config {
    static constexpr int D = D_, NT = NT_;
    static constexpr bool kInt8 = INT8_;
    static constexpr int kRows = 8 * NT;              // queries of an item
    static constexpr int kSteps = D / 16;             // k16 steps of a score, and 16-channel tiles of an output
    static constexpr int kPlane = D == 96 ? kUnit * 112 : kUnit * D;  // bytes of one plane of a unit in shared memory
    static constexpr int kStage = 2 * kPlane;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kMerge = kWarps * kRows * D * 4;
    static constexpr int kArea = kRing > kMerge ? kRing : kMerge;     // the ring doubles as the warps' merge area
    static constexpr int kOffInfo = kArea;                            // float4 [warps][stages]: K scale, log2 V scale, tokens
    static constexpr int kOffStat = kOffInfo + kWarps * kStages * 16; // float [warps][rows][4]: m, l, M
    static constexpr int kSmem = kOffStat + kWarps * kRows * 16;
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

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void wait_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
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

// Where 16-byte piece `piece` of token `token` stands in a plane of a stage: rows of 128 bytes, pieces rotated by xor so
// that the reads of eight rows (K) and of eight pieces of every second row (V) meet no bank twice; 64-byte rows go in pairs;
// 96-byte rows are padded to 112, which does the same for 4-byte reads.
template <int D>
__device__ __forceinline__ int place(int token, int piece) {
    if constexpr (D == 128) return token * 128 + ((piece ^ (token & 7)) << 4);
    if constexpr (D == 96) return token * 112 + (piece << 4);
    return (token >> 1) * 128 + (((((token & 1) << 2) | piece) ^ (((token >> 1) & 3) << 1)) << 4);
}

// The work of request r: queries (rows x group), visible tokens, and its share of the chunk list.
struct Request {
    int first, queries, tokens;  // first row, rows * group, tokens that its last row sees at most
    int before;                  // tokens ahead of its first row (may be negative)
    int tiles, chunks;
};
template <int ROWS>
__device__ __forceinline__ Request request_of(const BlockAttentionParams& p, int r) {
    Request q;
    q.first = p.v.query_start_loc[r];
    const int last = p.v.query_start_loc[r + 1], length = p.v.seq_lens[r];
    const int rows = max(0, min(last, p.num_rows) - q.first);
    q.queries = rows * p.group;
    q.tokens = max(0, min(length, p.max_len));
    q.before = length - (last - q.first);
    q.tiles = (q.queries + ROWS - 1) / ROWS;
    q.chunks = max(1, (q.tokens + kChunk - 1) / kChunk);
    return q;
}
__device__ __forceinline__ int64_t work_of(const BlockAttentionParams& p, const Request& q) {
    return static_cast<int64_t>(q.tiles) * p.v.kv_heads * q.chunks;
}

// Sum of all requests' work, and the sum of those before request `until`, or (until < 0) the request that chunk `at * span`
// falls into and the work before it.  All threads of the block take part.
struct Place {
    int64_t total, before, span;
    int request;
};
struct PlaceShared {
    int64_t warp_sums[kWarps];
    int64_t before;
    int request;
};
template <int ROWS>
__device__ __forceinline__ Place find_place(const BlockAttentionParams& p, PlaceShared& shared, int at, int until) {
    const int n = p.v.num_requests, each = (n + kThreads - 1) / kThreads;
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
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) running += shared.warp_sums[w];
        place.total += shared.warp_sums[w];
    }
    place.span = max(static_cast<int64_t>(p.min_span), (place.total + p.spans - 1) / p.spans);
    const int64_t target = at * place.span;
    const bool mine = until < 0 ? (running <= target && target < running + sum) : (lo <= until && until < hi);
    if (mine) {
        for (int r = lo; r < hi; ++r) {
            const int64_t one = work_of(p, request_of<ROWS>(p, r));
            if (until < 0 ? target < running + one : r == until) {
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
__global__ void __launch_bounds__(kThreads, C::NT == 1 ? 4 : 3) block_attention_kernel(const BlockAttentionParams p) {
    constexpr int D = C::D, NT = C::NT, kRows = C::kRows, kSteps = C::kSteps;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PlaceShared place_shared;
    const BlockView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int page_shift = v.page_tokens == 16 ? 4 : 5;
    pdl_wait();
    pdl_launch_dependents();
    const Place start = find_place<kRows>(p, place_shared, blockIdx.x, -1);
    int64_t at = blockIdx.x * start.span;
    const int64_t end = min(at + start.span, start.total);
    if (at >= end) return;
    int r = start.request;
    int64_t before = start.before;  // work ahead of request r
    Request q = request_of<kRows>(p, r);
    const int64_t plane_bytes = v.num_blocks * v.kv_heads * static_cast<int64_t>(v.page_tokens) * D;
    const int64_t plane_scales = v.num_blocks * v.kv_heads;
    uint8_t* ring = smem + warp * kStages * C::kStage;
    const uint32_t ring_address = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    float4* info = reinterpret_cast<float4*>(smem + C::kOffInfo) + warp * kStages;
    float* stats = reinterpret_cast<float*>(smem + C::kOffStat);

    while (at < end) {
        int64_t local = at - before;
        if (local >= work_of(p, q)) {  // on to the next request that has work (there is one: at < total)
            before += work_of(p, q);
            q = request_of<kRows>(p, ++r);
            continue;
        }
        const int item = static_cast<int>(local / q.chunks);
        const int chunk0 = static_cast<int>(local - static_cast<int64_t>(item) * q.chunks);
        const int chunk1 = static_cast<int>(min(static_cast<int64_t>(q.chunks), chunk0 + (end - at)));
        const int head = item % v.kv_heads, query0 = item / v.kv_heads * kRows;
        const int token_begin = chunk0 * kChunk, token_end = min(chunk1 * kChunk, q.tokens);
        const int all_units = (token_end - token_begin + kUnit - 1) / kUnit;
        const int units = all_units > warp ? (all_units - warp + kWarps - 1) / kWarps : 0;

        // page ids: lane i holds that of the warp's unit 32 w + i, one window ahead
        const int32_t* table = v.block_table + static_cast<int64_t>(r) * v.table_stride;
        auto window = [&](int first) {
            const int unit = first + lane;
            return unit < units ? table[(token_begin + (warp + unit * kWarps) * kUnit) >> page_shift] : -1;
        };
        int ids = window(0), ids_next = units > 32 ? window(32) : -1;
        auto produce = [&](int unit, int stage) {
            if (unit < units) {
                if ((unit & 31) == 0 && unit > 0) {
                    ids = ids_next;
                    ids_next = window(unit + 32);
                }
                const int id = __shfl_sync(kFullMask, ids, unit & 31);
                const int token0 = token_begin + (warp + unit * kWarps) * kUnit;
                const bool real = id >= 0 && id < v.num_blocks;
                const int count = real ? min(kUnit, token_end - token0) : 0;  // the rest is zero-filled
                const int64_t page = real ? static_cast<int64_t>(id) * v.kv_heads + head : 0;
                const uint8_t* from = v.codes + ((page << page_shift) + (token0 & (v.page_tokens - 1))) * D;
                const uint32_t to = ring_address + stage * C::kStage;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const int piece = i * 32 + lane, token = piece / (D / 16);
                    const int offset = place<D>(token, piece % (D / 16));
                    const bool in = token < count;
                    copy16(to + offset, from + piece * 16, in);
                    copy16(to + C::kPlane + offset, from + plane_bytes + piece * 16, in);
                }
                float* word = reinterpret_cast<float*>(info + stage);
                if (lane < 2) copy4(static_cast<uint32_t>(__cvta_generic_to_shared(word + lane)), v.scales + lane * plane_scales + page);
                if (lane == 2) word[2] = __int_as_float(count);
            }
            commit_copies();
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) produce(i, i);

        // this thread's query channels as fp16: query 8 n + g, the channels that its K words hold
        uint32_t qf[NT][kSteps][2];
        float factor[NT][2];   // score units of queries 8 n + 2 t + {0, 1}
        int limit[NT][2];      // tokens that they see
        int least = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int query = query0 + n * 8 + g;
            const bool real = query < q.queries;
            const int row = q.first + query / p.group, query_head = head * p.group + query % p.group;
            const uint16_t* from = static_cast<const uint16_t*>(p.query) + row * p.query_stride + query_head * D;
            uint32_t raw[kSteps][2];
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                // channels of step s: four of them, at 16 s + 4 t (D = 96) or inside this thread's D / 4 contiguous ones
                const int channel = D == 96 ? s * 16 + t * 4 : t * (D / 4) + s * 4;
                const uint2 two = real ? *reinterpret_cast<const uint2*>(from + channel) : make_uint2(0u, 0u);
                raw[s][0] = two.x;
                raw[s][1] = two.y;
            }
            uint32_t amax = 0u;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 f = activation2(raw[s][i], p.fp16);
                    const uint32_t a = __float_as_uint(f.x) & 0x7fffffffu, b = __float_as_uint(f.y) & 0x7fffffffu;
                    amax = max(amax, max(a < 0x7f800000u ? a : 0u, b < 0x7f800000u ? b : 0u));
                }
            }
            amax = max(amax, __shfl_xor_sync(kFullMask, amax, 1));
            amax = max(amax, __shfl_xor_sync(kFullMask, amax, 2));
            // the largest magnitude goes to [2^14, 2^15): exact for everything down to 2^-39 of it
            const int e = amax == 0u ? 0 : max(static_cast<int>(amax >> 23) - 127 - 14, -120);
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 f = activation2(raw[s][i], p.fp16);
                    qf[n][s][i] = pack_activation2(f.x * down, f.y * down, true);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                factor[n][i] = __shfl_sync(kFullMask, up, (2 * t + i) * 4) * p.scale_log2;
                const int column = query0 + n * 8 + 2 * t + i;
                limit[n][i] = column < q.queries ? max(0, min(q.tokens, q.before + column / p.group + 1)) : 0x7fffffff;
                least = min(least, limit[n][i]);
            }
        }
        least = __reduce_min_sync(kFullMask, least);

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

        int stage = 0, next = kStages - 1;
        for (int unit = 0; unit < units; ++unit) {
            wait_copies<kStages - 2>();
            __syncwarp();
            produce(unit + kStages - 1, next);
            const uint8_t* keys = ring + stage * C::kStage;
            const uint8_t* values = keys + C::kPlane;
            const float4 about = info[stage];
            next = stage;
            stage = stage + 1 == kStages ? 0 : stage + 1;
            const int token0 = token_begin + (warp + unit * kWarps) * kUnit;
            const int count = __float_as_int(about.z);

            // scores
            float x[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
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
                    low[s] = *reinterpret_cast<const uint32_t*>(keys + place<D>(g, s) + t * 4);
                    high[s] = *reinterpret_cast<const uint32_t*>(keys + place<D>(g + 8, s) + t * 4);
                }
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                uint32_t a[4];
                to_half<C::kInt8>(low[s], a[0], a[2]);
                to_half<C::kInt8>(high[s], a[1], a[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma(x[n], a, qf[n][s][0], qf[n][s][1]);
            }
            const float value_scale = log2_fast(about.y);
            const bool masked = count < kUnit || token0 + kUnit > least;
            bool raise = false;
            float top[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[n][i] *= about.x * factor[n][i & 1];
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
            if (p.scores != nullptr) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int column = query0 + n * 8 + 2 * t + (i & 1), token = token0 + g + (i >> 1) * 8;
                        if (column < q.queries && token < limit[n][i & 1]) {
                            const int row = q.first + column / p.group, query_head = head * p.group + column % p.group;
                            p.scores[(static_cast<int64_t>(row) * p.heads + query_head) * p.score_stride + token] = x[n][i];
                        }
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
            // weights; the value scale goes into the exponent
            uint32_t weight[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    l[n][i & 1] += exp2_fast(x[n][i] - m[n][i & 1]);
                    w[i] = exp2_fast(x[n][i] + (value_scale + kLift - M[n][i & 1]));
                }
                weight[n][0] = transpose8x8(pack_activation2(w[0], w[1], true));
                weight[n][1] = transpose8x8(pack_activation2(w[2], w[3], true));
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
                    for (int w = 0; w < kWords; ++w) word[i][w] = *reinterpret_cast<const uint32_t*>(values + token * 112 + g * 12 + w * 4);
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
                    for (int n = 0; n < NT; ++n) mma(o[2 * w + h][n], a, weight[n][0], weight[n][1]);
                }
            }
        }

        // ---- the warps' results are joined ----
        wait_copies<0>();
        __syncthreads();
        float* area = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int step = 4; step < 32; step <<= 1) l[n][i] += __shfl_xor_sync(kFullMask, l[n][i], step);
                const int column = n * 8 + 2 * t + i;
                float* to = area + (warp * kRows + column) * D + g * (D / 8);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) *reinterpret_cast<float2*>(to + 2 * s) = make_float2(o[s][n][i], o[s][n][i + 2]);
                if (g == 0) *reinterpret_cast<float4*>(stats + (warp * kRows + column) * 4) = make_float4(m[n][i], l[n][i], M[n][i], 0.f);
            }
        }
        __syncthreads();
        const bool whole = chunk0 == 0 && chunk1 == q.chunks;
        // a span leaves at most two unfinished pieces: the one at its start and the one at its end
        const int64_t slot = 2LL * blockIdx.x + (at > blockIdx.x * start.span ? 1 : 0);
        for (int piece = tid; piece < kRows * (D / 4); piece += kThreads) {
            const int column = piece / (D / 4), channel = piece % (D / 4) * 4;
            const int query = query0 + column;
            if (query >= q.queries) continue;
            float4 stat[kWarps];
            float m_all = kNever, M_all = kNever, l_all = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                stat[w] = *reinterpret_cast<const float4*>(stats + (w * kRows + column) * 4);
                m_all = fmaxf(m_all, stat[w].x);
                M_all = fmaxf(M_all, stat[w].z);
            }
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 part = *reinterpret_cast<const float4*>(area + (w * kRows + column) * D + channel);
                const float share = exp2_fast(stat[w].z - M_all);
                l_all += stat[w].y * exp2_fast(stat[w].x - m_all);
                sum.x += part.x * share;
                sum.y += part.y * share;
                sum.z += part.z * share;
                sum.w += part.w * share;
            }
            if (whole) {
                write_output(p, q.first + query / p.group, head * p.group + query % p.group, D, channel, sum, m_all, l_all, M_all);
            } else {
                float* to = p.partials + (slot * kRows + column) * C::kSlot;
                *reinterpret_cast<float4*>(to + channel) = sum;
                if (channel == 0) *reinterpret_cast<float4*>(to + D) = make_float4(m_all, l_all, M_all, 0.f);
            }
        }
        __syncthreads();
        at += chunk1 - chunk0;
    }
}

// Joins the pieces of the items that more than one span took part in: one CTA for each (row, query head).
template <typename C>
__global__ void __launch_bounds__(kThreads) block_join_kernel(const BlockAttentionParams p) {
    constexpr int D = C::D, kRows = C::kRows, kLanes = D / 4;
    __shared__ PlaceShared place_shared;
    __shared__ float4 sums[kWarps][kLanes];
    __shared__ float2 totals[kWarps], tops[kWarps];
    const BlockView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.heads, query_head = blockIdx.x % p.heads, head = query_head / p.group;
    pdl_wait();
    pdl_launch_dependents();
    const int r = find_request(v.query_start_loc, v.num_requests, row, lane);
    if (r >= v.num_requests) return;
    const Request q = request_of<kRows>(p, r);
    if (row < q.first || q.chunks == 1) return;
    const Place place = find_place<kRows>(p, place_shared, 0, r);
    const int query = (row - q.first) * p.group + query_head % p.group, column = query % kRows;
    const int64_t a = place.before + (static_cast<int64_t>(query / kRows) * v.kv_heads + head) * q.chunks, b = a + q.chunks;
    const int first = static_cast<int>(a / place.span), count = static_cast<int>((b - 1) / place.span) - first + 1;
    if (count == 1) return;
    auto part = [&](int i) -> const float* {
        const int64_t slot = 2LL * (first + i) + (i == 0 && a > first * place.span ? 1 : 0);
        return p.partials + (slot * kRows + column) * C::kSlot;
    };
    float m = kNever, M = kNever;
    for (int i = tid; i < count; i += kThreads) {
        const float4 stat = *reinterpret_cast<const float4*>(part(i) + D);
        m = fmaxf(m, stat.x);
        M = fmaxf(M, stat.z);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
        M = fmaxf(M, __shfl_xor_sync(kFullMask, M, o));
    }
    if (lane == 0) tops[warp] = make_float2(m, M);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        m = fmaxf(m, tops[w].x);
        M = fmaxf(M, tops[w].y);
    }
    float l = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = warp; i < count; i += kWarps) {
        const float* from = part(i);
        const float4 stat = *reinterpret_cast<const float4*>(from + D);
        const float share = exp2_fast(stat.z - M);
        l += stat.y * exp2_fast(stat.x - m);
        if (lane < kLanes) {
            const float4 x = *reinterpret_cast<const float4*>(from + lane * 4);
            sum.x += x.x * share;
            sum.y += x.y * share;
            sum.z += x.z * share;
            sum.w += x.w * share;
        }
    }
    if (lane < kLanes) sums[warp][lane] = sum;
    if (lane == 0) totals[warp] = make_float2(l, 0.f);
    __syncthreads();
    if (tid < kLanes) {
        l = 0.f;
        sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float4 x = sums[w][tid];
            l += totals[w].x;
            sum.x += x.x;
            sum.y += x.y;
            sum.z += x.z;
            sum.w += x.w;
        }
        write_output(p, row, query_head, D, tid * 4, sum, m, l, M);
    }
}

// Adds 2^(score - lse), summed over the rows and query heads of a KV head, to the weights: one thread for each token.
// One CTA adds to a token's weight in a call, so the sum's order is fixed; the atomic is for requests that share blocks.
__global__ void __launch_bounds__(kThreads) block_weights_kernel(const BlockAttentionParams p) {
    const BlockView& v = p.v;
    const int r = blockIdx.x / v.kv_heads, head = blockIdx.x % v.kv_heads;
    pdl_wait();
    pdl_launch_dependents();
    const Request q = request_of<8>(p, r);
    const int page_shift = v.page_tokens == 16 ? 4 : 5;
    for (int token = blockIdx.y * kThreads + threadIdx.x; token < q.tokens; token += gridDim.y * kThreads) {
        const int id = v.block_table[static_cast<int64_t>(r) * v.table_stride + (token >> page_shift)];
        if (id < 0 || id >= v.num_blocks) continue;
        float sum = 0.f;
        for (int query = 0; query < q.queries; ++query) {
            if (token > q.before + query / p.group) continue;
            const int64_t at = static_cast<int64_t>(q.first + query / p.group) * p.heads + head * p.group + query % p.group;
            sum += exp2_fast(p.scores[at * p.score_stride + token] - p.row_lse[at]);
        }
        if (sum != 0.f) atomicAdd(v.weights + ((static_cast<int64_t>(id) * v.kv_heads + head) << page_shift) + (token & (v.page_tokens - 1)), sum);
    }
}

template <int D, bool INT8, int NT>
cudaError_t launch(const BlockAttentionParams& p, cudaStream_t stream) {
    using C = Config<D, INT8, NT>;
    static std::atomic<uint64_t> prepared{0};  // devices whose shared-memory limit was raised
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if (C::kSmem > 48 * 1024 && (device >= 64 || !(prepared.load(std::memory_order_relaxed) >> device & 1))) {
        err = cudaFuncSetAttribute(block_attention_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (err != cudaSuccess) return err;
        if (device < 64) prepared.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    const bool programmatic = p.programmatic_launch != 0;
    err = launch_chained(block_attention_kernel<C>, p, dim3(static_cast<unsigned>(p.spans)), kThreads, C::kSmem, 1, programmatic, stream);
    if (err == cudaSuccess && p.max_len > kChunk)  // items of one chunk are never cut
        err = launch_chained(block_join_kernel<C>, p, dim3(static_cast<unsigned>(p.num_rows) * p.heads), kThreads, 0, 1, programmatic, stream);
    if (err == cudaSuccess && p.accumulate) {
        const unsigned parts = static_cast<unsigned>(std::min(64, (p.max_len + kThreads - 1) / kThreads));
        if (parts > 0)
            err = launch_chained(block_weights_kernel, p, dim3(static_cast<unsigned>(p.v.num_requests) * p.v.kv_heads, parts), kThreads, 0, 1,
                                 programmatic, stream);
    }
    return err;
}

template <int D, bool INT8>
cudaError_t launch_tiles(const BlockAttentionParams& p, cudaStream_t stream) {
    return p.query_tiles == 1 ? launch<D, INT8, 1>(p, stream) : launch<D, INT8, 2>(p, stream);
}

}  // namespace

int block_attention_slot_floats(int head_dim, int query_tiles) { return 8 * query_tiles * (head_dim + 4); }
int block_attention_chunk() { return kChunk; }

cudaError_t launch_block_attention(const BlockAttentionParams& p, int head_dim, int int8, cudaStream_t stream) {
    if (head_dim == 128) return int8 ? launch_tiles<128, true>(p, stream) : launch_tiles<128, false>(p, stream);
    if (head_dim == 96) return int8 ? launch_tiles<96, true>(p, stream) : launch_tiles<96, false>(p, stream);
    return int8 ? launch_tiles<64, true>(p, stream) : launch_tiles<64, false>(p, stream);
}

}  // namespace rq
