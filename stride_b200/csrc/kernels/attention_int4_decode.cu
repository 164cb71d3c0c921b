// Decode attention over a paged cache held in 4 bits (int4_cache.cuh), on the tensor cores.
//
// A single query reads every key of its request: the bytes of the cache bound it, 5 bits an entry. So that the work on an entry stays below
// the time its bytes take, an entry is never turned into a value: numbers go to the matrix instructions as they are, scales and centres are
// applied to scores and weights, of which there are 32 times fewer.
//
//   score(t) = sum_g s_tg (q_g . n_t) + (c_tg - 8 s_tg) sum q_g          out = sum_t (P_t s_tg) n_t + sum_t P_t (c_tg - 8 s_tg)
//
// * A number of 4 bits under the mask 0x000f000f (or 0x00f000f0) is a pair of 16-bit floating point numbers below the smallest normal one: n 2^-24
//   (or n 2^-20). Matrix instructions take those exactly, so one instruction unpacks two entries. The factors are powers of two: the query's
//   entries that meet the second kind are divided by 16 beforehand, the outputs of the second kind afterwards.
// * Keys are the A operand (16 tokens by 16 entries), the 8 columns of B are the group's query heads; the products of a group of 32 entries end in
//   an accumulator of their own, which the token's scale multiplies. Values are the A operand of the second product (16 entries by 16 tokens),
//   the weights P_t s_tg its B operand: a transpose of 8 x 8 in the warp.
// * Scales and centres themselves go through products in bfloat16, which they are exact in: with the sums of the query on the side of the keys,
//   with P on the side of the values, both in two parts, 16 bits. P s is rounded to 16 bits (2^-11 at most), so what the offset of 8 adds in
//   one product the other takes off but for that. The sum of the weights comes from the same product, from rows of ones.
// * The query is scaled by a power of two to below 2^15. The reference R of a weight 2^(score - R) is the running maximum of score + log2 of the
//   token's largest scale or centre, so that what is rounded to 16 bits lies below 2^8 and its largest near 1 whatever the values' size; R moves
//   only when a product passes 2^8 (a vote per tile), and then everything is rescaled.
// * What falls below 2^-24 is lost in 16-bit floating point, which a group does not notice whose own products reach near 1. The row that R comes
//   from vouches for them: where its smallest group is within a factor of 64 of its largest, every group has a product of 2^-6. Where it is not
//   (a value channel that stands out), the products of the second kind run in bfloat16, which has the range, with P s in two parts and the numbers
//   made whole, until R comes from a row that vouches for its groups again: 64 requests of such values take 121 us for 95.
//
// The work of a launch is a row of units, 128 keys of one (token, key head) each, in the order of tokens and key heads; every CTA takes an equal
// stretch of it (it works out from the positions where its own begins), so requests of any lengths keep all SMs busy to the end and a
// (token, key head) is cut only where a stretch ends. Parts of one are merged by the CTA that draws its last ticket, in the order of the keys.
//
// Measured: 64 requests of up to 8192 keys, 8 key heads of 128, group 4: 345 MB in 95 us, 3.6 TB/s, 0.56 of the copy rate; 8 requests 26 us; one
// request of 2048 keys 10.3 us. What bounds a full batch is the instructions between the copies and the products: 168 registers let three warps
// run on a scheduler, which issue in 0.51 of the cycles and wait for their own last instruction in most others; of a warp's cycles on 32
// keys 700 go to the scores, 350 to the softmax, 880 to the values, 230 to waiting for copies. Before the products in bfloat16 came beside those in 16-bit floating point
// it took 93; measured against that: whole units instead of equal stretches 97 us; cp.async instead of bulk copies 104; one ring for the CTA instead of one a warp 100; four CTAs an SM with two stages and four lanes
// asking for copies the same; P in one part instead of two 90, with an error of 2.4e-3 instead of 1.8e-3. One request is a chain of latencies:
// prologue 3.0 thousand cycles, the first pages and copies 3 to 5, a few tiles, the parts' sums 2.4, ticket and merge 3.5.
// A warp owns tiles of 32 keys and a ring of copies: a bulk copy for each 16 keys and one for their values where pages hold whole sixteens (a page's
// rows of one head lie side by side), 16- or 8-byte copies by all lanes otherwise.
#include "int4_cache.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"      // mbarrier helpers

namespace stride {
namespace four {

constexpr int kSub = 16;                // keys of half a tile: rows of a matrix instruction, and of a copy
constexpr int kTile = 2 * kSub;         // keys of a warp's tile
constexpr int kWarps = 4;
constexpr int kUnit = kTile * kWarps;   // keys that a CTA's warps cover with a tile each
constexpr int kStages = 3;
constexpr int kWindow = 16;             // tiles whose pages the lanes look up at once, a half each
constexpr int kTicketInts = 65536;      // ticket counters at the start of the scratch, one per (token, key head)
constexpr int kMostCtas = 148 * 3;      // of a launch: what fits at once
constexpr int kCodeBeyondBound = 32;    // as in attention_decode.cu
constexpr int kCodeCopyWait = 81;       // a wait for a tile's copies ran out
constexpr float kLimit = 256.f;         // what a weight's product with a scale may reach before R moves
constexpr float kMostWeight = 1.1529215e18f;    // 2^60, what a weight may (its product with a centre, below 2^64, stays a number)
constexpr float kMostUneven = 64.f;     // how far apart the groups of a row may be for 16-bit floating point
constexpr float kLeastLog = -90.f;      // log2 of the least size that R counts: a weight stays below 2^98

struct Decode {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    const uint8_t* k_pages;
    const uint8_t* v_pages;
    const int32_t* table;
    const int32_t* seq_of_token;
    const int32_t* positions;
    const float* sinks;
    const float* slopes;
    float* part_o;          // [2 CTAs][group][hd]: what a stretch holds of a (token, key head) that it shares with others
    float* part_ml;         // [2 CTAs][group][2]: R, sum of weights
    int* tickets;           // [token][key head]
    int* status;
    int q_stride, table_width, table_rows, num_pages, nq, nkv, page_size, window, tokens, max_context;
    float scale_log2e, cap_log2e, scale_over_cap;        // cap_log2e 0: no cap
};

// Whether a token reads keys: not a padded row, nor one of a request or position that the table or the launch's bound does not hold.
__device__ __forceinline__ bool reads(const Decode& a, int seq, int pos) { return seq >= 0 && seq < a.table_rows && pos >= 0 && pos < a.max_context; }
// The keys of a token in units: first unit and how many; none where it reads none.
struct Span {
    int first, units;
};
__device__ __forceinline__ Span span_of(const Decode& a, int t) {
    const int seq = a.seq_of_token[t], pos = a.positions[t];
    if (!reads(a, seq, pos)) return {0, 0};
    const int first = a.window > 0 ? max(0, pos - a.window + 1) / kUnit : 0;
    return {first, pos / kUnit - first + 1};
}

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
template <int BYTES>
__device__ __forceinline__ void small_copy(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
// D = A B + C, 16-bit floating point (or bfloat16) inputs, 32-bit accumulators.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2], float c0, float c1,
                                        float c2, float c3) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2], float c0, float c1,
                                         float c2, float c3) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// The transpose of an 8 x 8 matrix of 16-bit entries: lane l holds entries 2 (l % 4) and the next of row l / 4.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
__device__ __forceinline__ float exp2_quick(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int G>
__device__ __forceinline__ void load_words(uint32_t (&w)[G], const void* p) {       // G words from shared memory, 4 G bytes aligned
    if constexpr (G == 4) {
        const uint4 v = *static_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
        const uint2 v = *static_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    }
}
// The token of half a tile that stands in row r of the score tile: an order in which the lanes that read together find their rows in different banks
// (rows are 20 G bytes apart).
template <int G>
__device__ __forceinline__ int token_of(int r) {
    return G == 4 ? (r & 8) + (r & 1) * 4 + ((r & 7) >> 1) : (r & 3) * 4 + (r >> 2);
}
// The largest of the scales in a row's parameters (positive, or zero): as 16-bit integers, two at once, whatever the other halves hold.
template <int G>
__device__ __forceinline__ float largest_scale(const uint32_t (&p)[G]) {
    uint32_t m = p[0];
#pragma unroll
    for (int g = 1; g < G; ++g) m = __vmaxu2(m, p[g]);
    return bf16_low(m);
}
// log2 of the largest of a row's scales and its centres' sizes, 0 of them counted as 2^kLeastLog. uneven: some group's lies below it
// by more than kMostUneven, or all of it below 2^kLeastLog.
template <int G>
__device__ __forceinline__ float log2_size(const uint32_t (&p)[G], bool& uneven) {
    float m = 0.f, least = INFINITY;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float size = fmaxf(bf16_low(p[g]), fabsf(bf16_high(p[g])));
        m = fmaxf(m, size);
        least = fminf(least, size);
    }
    const float log2 = __log2f(m);
    uneven = !(least * kMostUneven >= m && log2 >= kLeastLog);
    return fmaxf(log2, kLeastLog);
}
// Two numbers in 16-bit halves under 0x000f000f, times `by` (a power of two up to 16), in bfloat16: 128 + n is exact there, and so are both steps.
__device__ __forceinline__ uint32_t whole_numbers(uint32_t n, float by) {
    const uint32_t biased = n | 0x43004300u;
    const __nv_bfloat162 y = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&biased), __float2bfloat162_rn(by), __float2bfloat162_rn(-128.f * by));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// G: groups of a head (head size 32 G). NT: tiles of 8 query heads.
template <int G, int NT, bool BULK>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) decode_kernel(const Decode a) {
    constexpr int HD = 32 * G, ROW = 20 * G, HALF = kSub * ROW, STAGE = 4 * HALF;      // a stage: the keys of either half, then their values
    pdl_trigger();
    pdl_wait();
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[kWarps][kStages];
    __shared__ uint32_t copied[kWarps][BULK ? 1 : kStages];         // small copies: the keys of a stage's tile that have a page, a bit each
    __shared__ int warp_sums[kWarps];
    __shared__ int begin_token, begin_units;
    __shared__ Span begin_span;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, group = a.nq / a.nkv;

    // ---- this CTA's stretch: `left` units from unit `skip` of (t, kvh) on
    int t = 0, kvh = 0, skip = 0, left = 0;
    long long total = 0, begin = 0, stretches = 0;
    {
        const int chunk = (a.tokens + kWarps * 32 - 1) / (kWarps * 32), t_lo = threadIdx.x * chunk, t_hi = min(a.tokens, t_lo + chunk);
        Span span = {0, 0};                                         // of the thread's last token
        int mine = 0;
        bool idle = false;                                          // a token without keys is among them
        for (int i = t_lo; i < t_hi; ++i) {
            span = span_of(a, i);
            mine += span.units;
            idle = idle || span.units == 0;
        }
        int upto = mine;                                            // with the lanes and warps before
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, s);
            if (lane >= s) upto += v;
        }
        if (lane == 31) warp_sums[warp] = upto;
        idle = __syncthreads_or(idle);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) upto += sum;
            sum += warp_sums[w];
        }
        total = static_cast<long long>(sum) * a.nkv;
        stretches = min(static_cast<long long>(gridDim.x), total);
        if (blockIdx.x < stretches) {
            if (total < (1LL << 31) / gridDim.x) {                  // 32-bit divisions, a tenth of the time
                begin = static_cast<uint32_t>(blockIdx.x) * static_cast<uint32_t>(total) / static_cast<uint32_t>(stretches);
                left = static_cast<int>((blockIdx.x + 1u) * static_cast<uint32_t>(total) / static_cast<uint32_t>(stretches) - static_cast<uint32_t>(begin));
            } else {
                begin = blockIdx.x * total / stretches;
                left = static_cast<int>((blockIdx.x + 1) * total / stretches - begin);
            }
            // units are counted token by token, key heads inside: the token whose heads hold unit `begin`
            if (begin < static_cast<long long>(upto) * a.nkv && begin >= static_cast<long long>(upto - mine) * a.nkv) {
                int before = upto - mine, i = t_lo;
                for (; chunk > 1; ++i) {
                    span = span_of(a, i);
                    if (begin < static_cast<long long>(before + span.units) * a.nkv) break;
                    before += span.units;
                }
                begin_token = i;
                begin_units = before;
                begin_span = span;
            }
        }
        __syncthreads();
        if (idle) {
            for (int i = blockIdx.x; i < a.tokens; i += gridDim.x) {        // rows without keys: zeros
                const int seq = a.seq_of_token[i], pos = a.positions[i];
                if (reads(a, seq, pos)) continue;
                for (int d = threadIdx.x; d < a.nq * HD; d += blockDim.x) a.out[static_cast<size_t>(i) * a.nq * HD + d] = __float2bfloat16_rn(0.f);
                if (seq >= 0 && threadIdx.x == 0) complain(a.status, seq < a.table_rows ? kCodeBeyondBound : kCodeNoPage);
            }
        }
    }
    if (left == 0) return;
    t = begin_token;
    long long item = static_cast<long long>(begin_units) * a.nkv;   // the first unit of (t, kvh)
    Span span = begin_span;
    kvh = static_cast<int>(begin - item) / span.units;
    item += static_cast<long long>(kvh) * span.units;
    skip = static_cast<int>(begin - item);
    auto stretch_of = [&](long long unit) {
        if (total < (1LL << 31) / gridDim.x)
            return static_cast<int>((static_cast<uint32_t>(unit + 1) * static_cast<uint32_t>(stretches) + static_cast<uint32_t>(total) - 1) / static_cast<uint32_t>(total)) - 1;
        return static_cast<int>(((unit + 1) * stretches + total - 1) / total - 1);
    };

    unsigned char* ring = smem + warp * kStages * STAGE;
    if (BULK) {
        if (lane == 0)
            for (int s = 0; s < kStages; ++s) tc::mbar_init(tc::smem_u32(&bars[warp][s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    const int row_a = token_of<G>(g), row_b = token_of<G>(g + 8);                                   // tokens of this lane's score rows
    const int col[4] = {token_of<G>(2 * c), token_of<G>(2 * c + 1), token_of<G>(2 * c + 8), token_of<G>(2 * c + 9)};        // of its weights
    const uint32_t pick = g < 4 ? 0x7632u : 0x5410u;            // rows of `cen`: centres or scales
    const bool bent = a.cap_log2e > 0.f || a.slopes != nullptr;
    bool alive = true;
    uint32_t uses = 0, held = 0;            // per stage: the parity of its barrier, and which halves of its tile were copied
    int stage = 0;

    for (;;) {          // ---- a (token, key head), or what the stretch holds of one
    const int n_tiles = min(left, span.units - skip), lo = (span.first + skip) * kUnit;
    const int pos = a.positions[t], first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int32_t* table = a.table + static_cast<size_t>(a.seq_of_token[t]) * a.table_width;
    auto tile_base = [&](int j) { return lo + j * kUnit + warp * kTile; };
    auto page_of = [&](int key) {
        const int index = key / a.page_size;
        return index < a.table_width ? table[index] : -1;
    };
    // the bytes at which a key's row of this head lies, or all ones where there is no such page
    auto row_at = [&](int key, int page) {
        if (page < 0 || page >= a.num_pages) {
            complain(a.status, kCodeNoPage);
            return ~size_t(0);
        }
        return ((static_cast<size_t>(page) * a.nkv + kvh) * a.page_size + key % a.page_size) * ROW;
    };
    // the query's rows, on their way beside the pages: lane (g, c) holds, of head 8 nt + g, entries 32 grp + 8 c .. + 7
    uint4 rows[NT][G];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
            const int head = 8 * nt + g;
            const __nv_bfloat16* src = a.q + static_cast<size_t>(t) * a.q_stride + static_cast<size_t>(kvh * group + head) * HD + 32 * grp + 8 * c;
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (head < group) {
                if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
                    raw = *reinterpret_cast<const uint4*>(src);
                } else {
                    const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
                    raw = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                }
            }
            rows[nt][grp] = raw;
        }
    // BULK: lane 2 i + h answers for half h of tile `window` + i: its row, and for the window after it the page
    size_t my_row = ~size_t(0);
    int my_page = -1;
    uint32_t live = 0;
    auto half_key = [&](int window) { return tile_base(window + (lane >> 1)) + (lane & 1) * kSub; };
    auto wanted = [&](int window) {
        const int key = half_key(window);
        return window + (lane >> 1) < n_tiles && key <= pos && key + kSub > first;
    };
    if (BULK && wanted(0)) my_page = page_of(half_key(0));
    auto issue = [&](int j, int stage) {
        if (j >= n_tiles) {
            if (!BULK) cp_async_commit();
            return;
        }
        if (BULK) {
            if (j % kWindow == 0) {
                my_row = wanted(j) ? row_at(half_key(j), my_page) : ~size_t(0);
                live = __ballot_sync(0xffffffffu, my_row != ~size_t(0));
                if (wanted(j + kWindow)) my_page = page_of(half_key(j + kWindow));
            }
            const uint32_t halves = live >> (2 * (j % kWindow)) & 3u;
            held = (held & ~(3u << (2 * stage))) | halves << (2 * stage);
            // (the barrier's one arrival, with the count of bytes, keeps the phase open whichever copy lands first)
            if ((lane >> 1) == j % kWindow && my_row != ~size_t(0)) {
                const uint32_t dst = tc::smem_u32(ring + stage * STAGE + (lane & 1) * HALF), bar = tc::smem_u32(&bars[warp][stage]);
                if ((lane & 1) == (halves == 2u)) tc::mbar_expect_tx(bar, halves == 3u ? 4 * HALF : 2 * HALF);
                if (halves == 3u && a.page_size % kTile == 0) {
                    if ((lane & 1) == 0) {
                        bulk_copy(dst, a.k_pages + my_row, 2 * HALF, bar);
                        bulk_copy(dst + 2 * HALF, a.v_pages + my_row, 2 * HALF, bar);
                    }
                } else {
                    bulk_copy(dst, a.k_pages + my_row, HALF, bar);
                    bulk_copy(dst + 2 * HALF, a.v_pages + my_row, HALF, bar);
                }
            }
            return;
        }
        const int base = tile_base(j);
        const uint32_t halves = (base <= pos && base + kSub > first ? 1u : 0u) | (base + kSub <= pos && base + kTile > first ? 2u : 0u);
        held = (held & ~(3u << (2 * stage))) | halves << (2 * stage);
        if (halves) {
            size_t row = ~size_t(0);
            const int key = base + lane;
            if (key >= first && key <= pos) row = row_at(key, page_of(key));
            const uint32_t have = __ballot_sync(0xffffffffu, row != ~size_t(0));
            if (lane == 0) copied[warp][stage] = have;
            unsigned char* to = ring + stage * STAGE;
#pragma unroll
            for (int i = 0; i < 5; ++i) {               // 32 rows of 5 pieces
                const int piece = i * 32 + lane, r = piece / 5, at = r * ROW + (piece - r * 5) * 4 * G;
                const size_t from = __shfl_sync(0xffffffffu, row, r);
                if (from != ~size_t(0)) {
                    small_copy<4 * G>(tc::smem_u32(to + at), a.k_pages + from + (piece - r * 5) * 4 * G);
                    small_copy<4 * G>(tc::smem_u32(to + 2 * HALF + at), a.v_pages + from + (piece - r * 5) * 4 * G);
                } else {
                    for (int b = 0; b < 4 * G; b += 4)
                        *reinterpret_cast<uint32_t*>(to + at + b) = *reinterpret_cast<uint32_t*>(to + 2 * HALF + at + b) = 0u;
                }
            }
        }
        cp_async_commit();
    };
    {
        int s = stage;
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
            issue(i, s);
            s = s + 1 == kStages ? 0 : s + 1;
        }
    }

    // ---- the query
    uint32_t qb[NT][G][2][2], cb[NT][2];            // B operands: of the numbers, of centres and scales
    float factor[NT][2], slope[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float x[G][8], most = 0.f;
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
            const uint4 raw = rows[nt][grp];
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[grp][i] = i & 1 ? bf16_high(w[i >> 1]) : bf16_low(w[i >> 1]);
                most = fmaxf(most, fabsf(x[grp][i]));
            }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // times 2^(up - 127), so that the largest entry lies in [2^14, 2^15); a query below 2^-112 keeps what 2^126 makes of it
        const int up = min(253, 268 - static_cast<int>(__float_as_uint(most) >> 23));
        const float by = __uint_as_float(static_cast<uint32_t>(up) << 23);
        float own = 0.f;
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[grp][i] *= by;
                sum += x[grp][i];
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (c == grp) own = sum * 5.9604644775390625e-08f;      // in the units of the numbers, 2^-24; lanes c >= G: no group, 0
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                qb[nt][grp][m][0] = pack_f16(x[grp][2 * m], x[grp][2 * m + 4]);
                qb[nt][grp][m][1] = pack_f16(x[grp][2 * m + 1] * 0.0625f, x[grp][2 * m + 5] * 0.0625f);
            }
        }
        {       // the sum in two parts of 8 bits, for the centre and, times -8, for the scale
            const float high = __bfloat162float(__float2bfloat16_rn(own));
            cb[nt][0] = pack_bf16(high, own - high);
            cb[nt][1] = pack_bf16(-8.f * high, -8.f * (own - high));
        }
        // (not 0, which would make masked scores no numbers)
        const float down = fmaxf(__uint_as_float(static_cast<uint32_t>(254 - up) << 23) * ((a.cap_log2e > 0.f ? a.scale_over_cap : a.scale_log2e) * 16777216.f),
                                 1.17549435e-38f);
        factor[nt][0] = __shfl_sync(0xffffffffu, down, 8 * c);
        factor[nt][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
#pragma unroll
        for (int e = 0; e < 2; ++e)
            slope[nt][e] = a.slopes != nullptr && 8 * nt + 2 * c + e < group ? a.slopes[kvh * group + 8 * nt + 2 * c + e] * 1.4426950408889634f : 0.f;
    }

    // cen: rows 0 .. G - 1 for the centres, from 4 on for the scales, 8 .. 15 (all alike) for the sum of the weights
    float R[NT][2], o[NT][G][2][4], cen[NT][4];
    uint32_t uneven_cols = 0;               // bit 2 nt + e: the row that R[nt][e] comes from is uneven (alike in all lanes of a column)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        R[nt][0] = R[nt][1] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            cen[nt][e] = 0.f;
#pragma unroll
            for (int grp = 0; grp < G; ++grp) o[nt][grp][0][e] = o[nt][grp][1][e] = 0.f;
        }
    }
    for (int j = 0; j < n_tiles; ++j) {
        const uint32_t halves = held >> (2 * stage) & 3u;
        if (BULK) {
            if (halves && alive) {
                alive = __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&bars[warp][stage]), uses >> stage & 1u, a.status, kCodeCopyWait));
                uses ^= 1u << stage;
            }
        } else {
            cp_async_wait<kStages - 1>();
            __syncwarp();
        }
        if (halves && alive) {
            const unsigned char* at = ring + stage * STAGE;
            const int base = tile_base(j);
            // some key of the tile is behind the token, before its window or without a page: what its row holds counts for nothing
            const uint32_t there = BULK ? ~0u : copied[warp][stage];
            const bool edge = halves != 3u || base + kTile - 1 > pos || base < first || there != ~0u;
            float x[NT][2][4], P[NT][2][4], amp[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned char* ks = at + h * HALF;
                uint32_t kw[2][G], kp[2][G];
                load_words<G>(kw[0], ks + row_a * ROW + c * 4 * G);
                load_words<G>(kw[1], ks + row_b * ROW + c * 4 * G);
                load_words<G>(kp[0], ks + row_a * ROW + 16 * G);
                load_words<G>(kp[1], ks + row_b * ROW + 16 * G);
                const uint32_t ca = *reinterpret_cast<const uint32_t*>(ks + row_a * ROW + 16 * G + 4 * (c % G)),
                               cc = *reinterpret_cast<const uint32_t*>(ks + row_b * ROW + 16 * G + 4 * (c % G));
                const uint32_t c0 = __byte_perm(ca, ca, 0x3232), c1 = __byte_perm(cc, cc, 0x3232), c2 = __byte_perm(ca, ca, 0x1010),
                               c3 = __byte_perm(cc, cc, 0x1010);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_bf16(x[nt][h], c0, c1, c2, c3, cb[nt], 0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int grp = 0; grp < G; ++grp) {
                    const uint32_t w0 = kw[0][grp], w1 = kw[1][grp], u0 = w0 >> 8, u1 = w1 >> 8;
                    const float s0 = bf16_low(kp[0][grp]), s1 = bf16_low(kp[1][grp]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float acc[4];
                        mma_f16(acc, w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, qb[nt][grp][0], 0.f, 0.f, 0.f, 0.f);
                        mma_f16(acc, u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, qb[nt][grp][1], acc[0], acc[1], acc[2], acc[3]);
                        x[nt][h][0] = fmaf(s0, acc[0], x[nt][h][0]);
                        x[nt][h][1] = fmaf(s0, acc[1], x[nt][h][1]);
                        x[nt][h][2] = fmaf(s1, acc[2], x[nt][h][2]);
                        x[nt][h][3] = fmaf(s1, acc[3], x[nt][h][3]);
                    }
                }
                uint32_t vp[2][G];
                load_words<G>(vp[0], ks + 2 * HALF + row_a * ROW + 16 * G);
                load_words<G>(vp[1], ks + 2 * HALF + row_b * ROW + 16 * G);
                amp[h][0] = largest_scale<G>(vp[0]);
                amp[h][1] = largest_scale<G>(vp[1]);
            }
            // where something bends the score, x becomes the score in units of log2 here; else it stays as it is, `unit` of them
            float unit[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) unit[nt][e] = bent ? 1.f : factor[nt][e];
            if (bent) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float y = x[nt][h][e] * factor[nt][e & 1];
                            if (a.cap_log2e > 0.f) y = a.cap_log2e * tanh_quick(y);
                            x[nt][h][e] = fmaf(slope[nt][e & 1], static_cast<float>(base + h * kSub + (e < 2 ? row_a : row_b) - pos), y);
                        }
            }
            uint32_t seen = 0xfu;           // of the score rows: half 0 row_a, row_b, half 1 row_a, row_b
            if (edge) {
                seen = 0u;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int key = base + h * kSub + (r ? row_b : row_a);
                        const bool ok = (halves >> h & 1u) && key <= pos && key >= first && (there >> (key - base) & 1u);
                        seen |= ok ? 1u << (2 * h + r) : 0u;
                        if (!ok) {
                            amp[h][r] = 0.f;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) x[nt][h][2 * r] = x[nt][h][2 * r + 1] = -INFINITY;
                        }
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float most_of[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) P[nt][h][e] = exp2_quick(fmaf(x[nt][h][e], unit[nt][e & 1], -R[nt][e & 1]));
                    most_of[h][0] = fmaxf(P[nt][h][0], P[nt][h][1]);
                    most_of[h][1] = fmaxf(P[nt][h][2], P[nt][h][3]);
                }
                const float product = fmaxf(fmaxf(most_of[0][0] * amp[0][0], most_of[0][1] * amp[0][1]),
                                            fmaxf(most_of[1][0] * amp[1][0], most_of[1][1] * amp[1][1]));
                const float weight = fmaxf(fmaxf(most_of[0][0], most_of[0][1]), fmaxf(most_of[1][0], most_of[1][1]));
                // (R is -inf until a tile with a key; then weights are infinite or, of masked keys, no numbers)
                if (__any_sync(0xffffffffu, !(product <= kLimit && weight <= kMostWeight))) {
                    float size[2][2];
                    bool uneven[2][2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t vp[2][G];
                        load_words<G>(vp[0], at + (2 + h) * HALF + row_a * ROW + 16 * G);
                        load_words<G>(vp[1], at + (2 + h) * HALF + row_b * ROW + 16 * G);
                        size[h][0] = log2_size<G>(vp[0], uneven[h][0]);
                        size[h][1] = log2_size<G>(vp[1], uneven[h][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float most = -INFINITY;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                most = x[nt][h][2 * r + e] == -INFINITY ? most : fmaxf(most, fmaf(x[nt][h][2 * r + e], unit[nt][e], size[h][r]));
#pragma unroll
                        for (int s = 4; s < 32; s <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
                        bool from_uneven = false;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                from_uneven = from_uneven || (uneven[h][r] && fmaf(x[nt][h][2 * r + e], unit[nt][e], size[h][r]) >= most);
                        const uint32_t lanes = __ballot_sync(0xffffffffu, from_uneven) & 0x11111111u << c, bit = 1u << (2 * nt + e);
                        if (most > R[nt][e] && 8 * nt + 2 * c + static_cast<int>(e) < group) uneven_cols = lanes ? uneven_cols | bit : uneven_cols & ~bit;
                        // (the weights' sum goes down in two steps: their values' sizes are in R, and the factor may be below any number)
                        const float next = fmaxf(R[nt][e], most), half = R[nt][e] == -INFINITY ? 0.f : exp2_quick(0.5f * (R[nt][e] - next)), by = half * half;
                        R[nt][e] = next;
                        cen[nt][e] *= by;
                        cen[nt][e + 2] = cen[nt][e + 2] * half * half;
#pragma unroll
                        for (int grp = 0; grp < G; ++grp)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                o[nt][grp][h][e] *= by;
                                o[nt][grp][h][e + 2] *= by;
                            }
                        // (-inf: the column has seen no key, or only such as are no numbers, which the weights then are, too)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int r = 0; r < 2; ++r) P[nt][h][2 * r + e] = exp2_quick(fmaf(x[nt][h][2 * r + e], unit[nt][e], next == -INFINITY ? 0.f : -next));
                    }
                }
            }
            const bool wide = __any_sync(0xffffffffu, uneven_cols != 0u);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned char* vs = at + (2 + h) * HALF;
                uint32_t vp[2][G], vw[4][G / 2], vc[4];
                load_words<G>(vp[0], vs + row_a * ROW + 16 * G);
                load_words<G>(vp[1], vs + row_b * ROW + 16 * G);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (G == 4) {
                        const uint2 v = *reinterpret_cast<const uint2*>(vs + col[i] * ROW + g * 2 * G);
                        vw[i][0] = v.x;
                        vw[i][1] = v.y;
                    } else {
                        vw[i][0] = *reinterpret_cast<const uint32_t*>(vs + col[i] * ROW + g * 2 * G);
                    }
                    vc[i] = *reinterpret_cast<const uint32_t*>(vs + col[i] * ROW + 16 * G + 4 * (g % G));
                }
                if (edge) {
#pragma unroll
                    for (int grp = 0; grp < G; ++grp) {
                        if (!(seen >> (2 * h) & 1u)) vp[0][grp] = 0u;
                        if (!(seen >> (2 * h + 1) & 1u)) vp[1][grp] = 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = base + h * kSub + col[i];
                        if (!(halves >> h & 1u) || key > pos || key < first || !(there >> (key - base) & 1u)) vc[i] = 0u;
                    }
                }
                const uint32_t a0 = __byte_perm(vc[0], vc[1], pick), a2 = __byte_perm(vc[2], vc[3], pick);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float rest[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) rest[e] = P[nt][h][e] - bf16_high(__float_as_uint(P[nt][h][e]));
                    const uint32_t high[2] = {transposed(__byte_perm(__float_as_uint(P[nt][h][0]), __float_as_uint(P[nt][h][1]), 0x7632)),
                                              transposed(__byte_perm(__float_as_uint(P[nt][h][2]), __float_as_uint(P[nt][h][3]), 0x7632))};
                    const uint32_t low[2] = {transposed(pack_bf16(rest[0], rest[1])), transposed(pack_bf16(rest[2], rest[3]))};
                    float(&d)[4] = cen[nt];
                    mma_bf16(d, a0, 0x3f803f80u, a2, 0x3f803f80u, high, d[0], d[1], d[2], d[3]);
                    mma_bf16(d, a0, 0x3f803f80u, a2, 0x3f803f80u, low, d[0], d[1], d[2], d[3]);
                }
                if (wide) {                         // P s 2^-24 in two parts of 8 bits beside whole numbers: the same units
#pragma unroll
                    for (int grp = 0; grp < G; ++grp) {
                        const uint32_t x0 = __byte_perm(vw[0][grp >> 1], vw[1][grp >> 1], grp & 1 ? 0x7632 : 0x5410),
                                       x1 = __byte_perm(vw[2][grp >> 1], vw[3][grp >> 1], grp & 1 ? 0x7632 : 0x5410), y0 = x0 >> 8, y1 = x1 >> 8;
                        const float s0 = bf16_low(vp[0][grp]), s1 = bf16_low(vp[1][grp]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float y[4] = {P[nt][h][0] * s0 * 5.9604644775390625e-08f, P[nt][h][1] * s0 * 5.9604644775390625e-08f,
                                                P[nt][h][2] * s1 * 5.9604644775390625e-08f, P[nt][h][3] * s1 * 5.9604644775390625e-08f};
                            float rest[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) rest[e] = y[e] - bf16_high(__float_as_uint(y[e]));
                            const uint32_t parts[2][2] = {{transposed(__byte_perm(__float_as_uint(y[0]), __float_as_uint(y[1]), 0x7632)),
                                                           transposed(__byte_perm(__float_as_uint(y[2]), __float_as_uint(y[3]), 0x7632))},
                                                          {transposed(pack_bf16(rest[0], rest[1])), transposed(pack_bf16(rest[2], rest[3]))}};
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint32_t u0 = k ? y0 : x0, u1 = k ? y1 : x1;
                                const uint32_t n0 = whole_numbers(u0 & 0x000f000fu, 1.f), n1 = whole_numbers(u0 >> 4 & 0x000f000fu, 16.f),
                                               n2 = whole_numbers(u1 & 0x000f000fu, 1.f), n3 = whole_numbers(u1 >> 4 & 0x000f000fu, 16.f);
                                float(&d)[4] = o[nt][grp][k];
                                mma_bf16(d, n0, n1, n2, n3, parts[0], d[0], d[1], d[2], d[3]);
                                mma_bf16(d, n0, n1, n2, n3, parts[1], d[0], d[1], d[2], d[3]);
                            }
                        }
                    }
                    continue;
                }
#pragma unroll
                for (int grp = 0; grp < G; ++grp) {
                    const uint32_t x0 = __byte_perm(vw[0][grp >> 1], vw[1][grp >> 1], grp & 1 ? 0x7632 : 0x5410),
                                   x1 = __byte_perm(vw[2][grp >> 1], vw[3][grp >> 1], grp & 1 ? 0x7632 : 0x5410), y0 = x0 >> 8, y1 = x1 >> 8;
                    const float s0 = bf16_low(vp[0][grp]), s1 = bf16_low(vp[1][grp]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint32_t b[2] = {transposed(pack_f16(P[nt][h][0] * s0, P[nt][h][1] * s0)),
                                               transposed(pack_f16(P[nt][h][2] * s1, P[nt][h][3] * s1))};
                        float(&d)[4] = o[nt][grp][0];
                        float(&f)[4] = o[nt][grp][1];
                        mma_f16(d, x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu, x1 & 0x00f000f0u, b, d[0], d[1], d[2], d[3]);
                        mma_f16(f, y0 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u, b, f[0], f[1], f[2], f[3]);
                    }
                }
            }
        }
        __syncwarp();           // every lane is done with the stage before it is refilled
        issue(j + kStages, stage);
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }

    // ---- the warps' results side by side in shared memory (the rings are no longer needed)
    const int before = stretch_of(item), parts = stretch_of(item + span.units - 1) - before + 1;
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);
    constexpr int RS = HD + 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int head = 8 * nt + 2 * c + e;
            float* dst = red + (warp * group + head) * RS;
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                const float centre = __shfl_sync(0xffffffffu, cen[nt][e], 4 * grp + c) - 8.f * __shfl_sync(0xffffffffu, cen[nt][e], 4 * (4 + grp) + c);
                if (head < group) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        dst[32 * grp + 4 * g + 2 * h] = fmaf(o[nt][grp][h][e], 16777216.f, centre);
                        dst[32 * grp + 4 * g + 2 * h + 1] = fmaf(o[nt][grp][h][e + 2], 1048576.f, centre);
                    }
                }
            }
            if (head < group && g == 0) {
                dst[HD] = R[nt][e];
                dst[HD + 1] = cen[nt][e + 2];
            }
        }
    __syncthreads();
    __nv_bfloat16* out = a.out + (static_cast<size_t>(t) * a.nq + kvh * group) * HD;
    // where a part lies: one that begins with the keys in the CTA's second place (it is its last), any other in its first
    auto place = [&](int part) { return static_cast<size_t>(2 * (before + part) + (part == 0)) * group; };
    for (int idx = threadIdx.x; idx < group * HD; idx += blockDim.x) {
        const int row = idx / HD, d = idx - row * HD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, red[(w * group + row) * RS + HD]);
        float acc = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float* src = red + (w * group + row) * RS;
            const float half = mm == -INFINITY ? 0.f : exp2f(0.5f * (src[HD] - mm));       // a warp without keys has weight 0
            acc += half * half * src[d];
            sum += src[HD + 1] * half * half;
        }
        if (parts == 1) {
            if (a.sinks != nullptr && mm != -INFINITY) sum += exp2f(fmaf(a.sinks[kvh * group + row], 1.4426950408889634f, -mm));
            out[idx] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc / sum);      // 0: no key had a page
            continue;
        }
        const size_t at = place(blockIdx.x - before) + row;
        a.part_o[at * HD + d] = acc;
        if (d == 0) {
            a.part_ml[at * 2] = mm;
            a.part_ml[at * 2 + 1] = sum;
        }
    }
    if (parts > 1) {
        // ---- the CTA that finishes last for this (token, key head) merges the parts
        __shared__ int is_last;
        __syncthreads();
        if (threadIdx.x == 0) {             // (the barriers order the CTA's stores before this thread's release, and its loads behind its acquire)
            int* ticket = a.tickets + static_cast<size_t>(t) * a.nkv + kvh;
            int drawn;
            asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(drawn) : "l"(ticket) : "memory");
            is_last = drawn == parts - 1;
            if (is_last) *ticket = 0;       // ready for the next launch; nobody else touches it before then
        }
        __syncthreads();
        if (is_last) {
            // a warp a head works out the weights, then a thread sums four columns, many parts on their way at once
            float* weights = reinterpret_cast<float*>(smem);        // [group][parts], then [group] sums
            for (int row = warp; row < group; row += kWarps) {
                float most = -INFINITY;
                for (int i = lane; i < parts; i += 32) {
                    const float v = __ldcg(a.part_ml + (place(i) + row) * 2);
                    weights[row * parts + i] = v;
                    most = fmaxf(most, v);
                }
                most = warp_max(most);
                float sum = 0.f;
                for (int i = lane; i < parts; i += 32) {
                    const float half = most == -INFINITY ? 0.f : exp2f(0.5f * (weights[row * parts + i] - most));
                    weights[row * parts + i] = half * half;
                    sum += __ldcg(a.part_ml + (place(i) + row) * 2 + 1) * half * half;
                }
                sum = warp_sum(sum);
                if (a.sinks != nullptr && most != -INFINITY) sum += exp2f(fmaf(a.sinks[kvh * group + row], 1.4426950408889634f, -most));
                if (lane == 0) weights[group * parts + row] = sum;
            }
            __syncthreads();
            for (int idx = threadIdx.x; idx < group * (HD / 4); idx += blockDim.x) {
                const int row = idx / (HD / 4), d = (idx - row * (HD / 4)) * 4;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 16
                for (int i = 0; i < parts; ++i) {
                    const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_o + (place(i) + row) * HD + d));
                    const float w = weights[row * parts + i];
                    acc.x = fmaf(w, v.x, acc.x);
                    acc.y = fmaf(w, v.y, acc.y);
                    acc.z = fmaf(w, v.z, acc.z);
                    acc.w = fmaf(w, v.w, acc.w);
                }
                const float sum = weights[group * parts + row];
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
                if (reinterpret_cast<uintptr_t>(a.out) % 8 == 0) {
                    *reinterpret_cast<uint2*>(out + row * HD + d) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[row * HD + d + i] = __float2bfloat16_rn(y[i]);
                }
            }
        }
    }
    // ---- on to the next
    left -= n_tiles;
    if (left == 0) return;
    item += span.units;
    skip = 0;
    if (++kvh == a.nkv) {
        kvh = 0;
        do span = span_of(a, ++t);
        while (span.units == 0);
    }
    tc::fence_proxy_async();        // the ring was written through the generic proxy: before the next copies into it
    __syncthreads();
    }
}

// CTAs of a launch: as many as fit at once, no more than there can be units.
inline int choose_ctas(int tokens, int nkv, int max_context, int group) {
    const long long units = static_cast<long long>(tokens) * nkv * ((static_cast<long long>(max_context) + kUnit - 1) / kUnit);
    const int fit = group <= 8 ? kMostCtas : 148 * 2;
    return units < fit ? static_cast<int>(units) : fit;
}

template <int G, int NT>
int launch_decode(const Decode& a, int ctas, cudaStream_t stream) {
    constexpr int smem = kWarps * kStages * 2 * kTile * 20 * G;        // 61 KB at head size 128
    static_assert(kWarps * 8 * NT * (32 * G + 2) * 4 <= smem && 8 * NT * (kMostCtas + 1) * 4 <= smem, "the warps' results and the parts' weights fit into the rings");
    // bulk copies: whole sixteens of keys side by side, from addresses that are multiples of 16 (rows of 40 bytes need not lie so)
    const bool bulk = a.page_size % kSub == 0 && (reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) % 16 == 0;
    cudaError_t e = allow_shared<decode_kernel<G, NT, true>>(smem);
    if (e == cudaSuccess) e = allow_shared<decode_kernel<G, NT, false>>(smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (bulk)
        stride::launch(decode_kernel<G, NT, true>, dim3(ctas), dim3(kWarps * 32), smem, stream, a);
    else
        stride::launch(decode_kernel<G, NT, false>, dim3(ctas), dim3(kWarps * 32), smem, stream, a);
    return STRIDE_LAUNCH_STATUS();
}

}  // namespace four
}  // namespace stride

using namespace stride;

extern "C" {

// Number of float32 scratch elements the launcher needs for these sizes.
long long stride_decode_int4_scratch_floats(int tokens, int nq, int nkv, int hd, int max_context) {
    if (tokens <= 0 || nq <= 0 || nkv <= 0 || max_context <= 0) return 0;
    const int group = nq / nkv;
    return four::kTicketInts + 2LL * four::choose_ctas(tokens, nkv, max_context, group) * group * (hd + 2);
}

struct DecodeCall {
    const __nv_bfloat16* q;         // [tokens, q_stride] with head h at columns [h hd, (h + 1) hd)
    __nv_bfloat16* out;             // [tokens, nq hd]
    const uint8_t* k_pages;         // [num_pages, nkv, page_size, 20 hd / 32]
    const uint8_t* v_pages;
    const int32_t* block_table;     // [requests, table_width]
    const int32_t* seq_of_token;
    const int32_t* positions;
    float* scratch;
    const float* sinks;
    const float* slopes;
    int* status;
    cudaStream_t stream;
    long long scratch_floats;
    int q_stride, num_pages, table_width, table_rows, tokens, nq, nkv, hd, page_size, window, max_context;
    float scale, softcap;
    int unused;
};

static_assert(sizeof(DecodeCall) == 160, "the record that the caller packs");

// One query token per row. `scratch` must be zero when it is first used (every launch leaves its tickets zero) and belongs to one stream at a
// time. A row whose position does not lie below `max_context` gets zeros, and code 32 in the status word; a key whose page is none of the
// cache's is left out, with code 33. Returns -2 for sizes it does not run: head sizes other than 64 and 128, groups above 16, more than
// 65536 (token, key head) pairs, pages at addresses that are no multiples of hd / 8.
int stride_decode_int4(const void* record) {
    const DecodeCall r = read_record<DecodeCall>(record);
    if (r.tokens < 0 || r.nq <= 0 || r.nkv <= 0 || r.page_size <= 0 || r.table_width <= 0 || r.table_rows <= 0 || r.num_pages <= 0 || r.window < 0 || r.softcap < 0.f ||
        r.max_context <= 0 || r.nq % r.nkv || r.status == nullptr)
        return STRIDE_BAD_ARGUMENT;
    if ((r.hd != 64 && r.hd != 128) || r.nq / r.nkv > 16 || r.max_context > (1 << 30)) return STRIDE_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(r.k_pages) | reinterpret_cast<uintptr_t>(r.v_pages)) % (r.hd / 8) || reinterpret_cast<uintptr_t>(r.scratch) % 16)
        return STRIDE_UNSUPPORTED;                      // (the pieces that small copies take of a row)
    if (r.tokens == 0) return 0;
    if (static_cast<long long>(r.tokens) * r.nkv > four::kTicketInts) return STRIDE_UNSUPPORTED;
    // units are counted in 32 bits token by token
    if (static_cast<long long>(r.tokens) * (r.max_context / four::kUnit + 1) > 2147483647LL) return STRIDE_UNSUPPORTED;
    if (r.scratch == nullptr || r.scratch_floats < stride_decode_int4_scratch_floats(r.tokens, r.nq, r.nkv, r.hd, r.max_context))
        return STRIDE_BAD_ARGUMENT;
    const int ctas = four::choose_ctas(r.tokens, r.nkv, r.max_context, r.nq / r.nkv);
    static_assert(sizeof(int) == sizeof(float), "the tickets live in the float scratch");
    four::Decode a;
    a.q = r.q;
    a.out = r.out;
    a.k_pages = r.k_pages;
    a.v_pages = r.v_pages;
    a.table = r.block_table;
    a.seq_of_token = r.seq_of_token;
    a.positions = r.positions;
    a.sinks = r.sinks;
    a.slopes = r.slopes;
    a.tickets = reinterpret_cast<int*>(r.scratch);
    a.part_o = r.scratch + four::kTicketInts;
    a.part_ml = a.part_o + 2LL * ctas * (r.nq / r.nkv) * r.hd;
    a.status = r.status;
    a.q_stride = r.q_stride;
    a.table_width = r.table_width;
    a.table_rows = r.table_rows;
    a.num_pages = r.num_pages;
    a.nq = r.nq;
    a.nkv = r.nkv;
    a.page_size = r.page_size;
    a.window = r.window;
    a.tokens = r.tokens;
    a.max_context = r.max_context;
    a.scale_log2e = r.scale * 1.4426950408889634f;
    a.cap_log2e = r.softcap * 1.4426950408889634f;
    a.scale_over_cap = r.softcap > 0.f ? r.scale / r.softcap : 0.f;
    const bool wide = r.nq / r.nkv > 8;
    if (r.hd == 64) return wide ? four::launch_decode<2, 2>(a, ctas, r.stream) : four::launch_decode<2, 1>(a, ctas, r.stream);
    return wide ? four::launch_decode<4, 2>(a, ctas, r.stream) : four::launch_decode<4, 1>(a, ctas, r.stream);
}

}  // extern "C"
