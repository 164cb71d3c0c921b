// Attention over a paged cache held in 4 bits (int4_cache.cuh): the exact kernel.
//
// The rule is that of attention_generic.cu, the numbers are those the rows stand for: softmax(q k^T scale) v over the keys j <= p (and
// j > p - window), scores capped at c tanh(s / c), a penalty slope_h (p - j), a sink per head in the denominator. Key j
// belongs to stream j / 32 % 8: a stream is an online softmax in 32 bits over its keys in order, 32 at a time, and a row's streams are
// joined in order. So every sum depends on p alone: a token's result has the same bits in a whole prompt, in a portion or alone, on
// whatever pages, and eight CTAs can work on a row at once.
//
// Tensor cores have no 32-bit products, so the 4 hd operations a row, head and key go through the FMA units. What bounds a long prompt is shared
// memory: every key is read from it once a warp, for the warp's rows. 2048 rows of 32 heads of 128 take 2.28 ms, 15 TFLOP/s. A few rows are
// bound by the chain of their keys: 2 portions of 50 rows at 1000 keys, 12 heads of 64, 38 us (103 without the streams side by side), one row
// at 8000 keys 110 us (707).
#include "int4_cache.cuh"

namespace stride {

constexpr int kStreams = 8, kStretch = 32, kRound = kStreams * kStretch;

// The first key of a stream at or behind the stretch that holds `key`, and its keys from there, counted from 0.
__device__ __forceinline__ int stream_begin(int key, int stream) {
    const int stretch = key / kStretch;
    return (stretch + (stream + kStreams - stretch % kStreams) % kStreams) * kStretch;
}
__device__ __forceinline__ int stream_key(int begin, int index) { return begin + index / kStretch * kRound + index % kStretch; }

// Joins a stream (m, l, acc) to those before it; -inf: it has seen no number.
template <int N>
__device__ __forceinline__ void join(float& M, float& L, float (&A)[N], float m, float l, const float (&acc)[N]) {
    const float next = fmaxf(M, m), a = M == -INFINITY ? 0.f : expf(M - next), b = m == -INFINITY ? 0.f : expf(m - next);
    L = __fadd_rn(__fmul_rn(L, a), __fmul_rn(l, b));
#pragma unroll
    for (int i = 0; i < N; ++i) A[i] = __fadd_rn(__fmul_rn(A[i], a), __fmul_rn(acc[i], b));
    M = next;
}

// The positions that the kernels count to: what lies ahead of the last key still fits 32 bits.
constexpr long long kMaxPositions = (1ll << 31) - (1ll << 14);

// The request of a row: -1 for a padded one, and for one whose request or position the block table does not hold (the status word says so).
__device__ __forceinline__ int request_of(int seq, int pos, int table_rows, int table_width, int page_size, int* status) {
    if (seq < 0) return -1;
    if (seq < table_rows && pos >= 0 && pos < min(static_cast<long long>(table_width) * page_size, kMaxPositions)) return seq;
    four::complain(status, four::kCodeNoPage);
    return -1;
}

// 32 keys and values at a time lie in shared memory as the numbers they stand for: one CTA, or a cluster of eight, one a stream, owns TQ consecutive
// rows and up to kTileHeads query heads of one key head, a warp NR of those (row, head) pairs. A key is taken apart once for all of them
// instead of once each, and what the next 32 hold is on its way while these are worked through. The streams of a pair meet in the shared
// memory of one of the CTAs, each of which joins an eighth of the pairs.
__device__ __forceinline__ void store_cluster(uint32_t local, uint32_t rank, float x) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(x) : "memory");
}
constexpr int kTileHeads = 4;

template <typename T, int G, int TQ, int NW, int NR, int CTAS>
__global__ void __launch_bounds__(NW * 32)
attention_int4_tile_kernel(const T* __restrict__ q, int q_stride, T* __restrict__ out, const uint8_t* __restrict__ k_pages,
                           const uint8_t* __restrict__ v_pages, int num_pages, const int32_t* __restrict__ block_table, int table_rows, int table_width,
                           const int32_t* __restrict__ seq_of_token, const int32_t* __restrict__ positions, int tokens, int nq, int nkv, int hd,
                           int page_size, float scale, int window, float softcap, const float* __restrict__ sinks, const float* __restrict__ slopes,
                           int* status) {
    static_assert(NW * NR == TQ * kTileHeads, "a pair of row and head for every place");
    static_assert(CTAS == 1 || CTAS == kStreams, "a CTA for all streams or for one");
    constexpr int OWN = (NW * NR + kStreams - 1) / kStreams;        // pairs that one of eight joins: pair i is CTA i % 8's
    constexpr int THREADS = NW * 32, KW = (32 * 4 * G + THREADS - 1) / THREADS, VW = (32 * 8 * G + THREADS - 1) / THREADS;       // words, half words a thread
    extern __shared__ __align__(16) float tile[];
    __shared__ size_t row_at[2][THREADS];               // where the rows of THREADS keys lie, and of those after them; all ones for none
    __shared__ float4 weights[NW * NR][8];              // of a pair's 32 keys
    __shared__ float joined[kStreams][CTAS > 1 ? OWN : 1][CTAS > 1 ? 32 * G + 2 : 1]; // what the streams made of this CTA's pairs: sums, maximum, sum of weights
    if (CTAS > 1) cluster_arrive();
    // (no early start for the next kernel: its waiting CTAs would take the places of this one's, which run for long and are few)
    pdl_wait();
    constexpr int width = 32 * G, kld = width + 4, bytes = 20 * G;
    float* const ks = tile;                             // [32][width + 4]
    float* const vs = ks + 32 * kld;                    // [32][width]
    float* const qs = vs + 32 * width;                  // [NW * NR][width]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = nq / nkv, parts = (group + kTileHeads - 1) / kTileHeads;
    const int rank = blockIdx.z, kvh = blockIdx.y / parts, head0 = kvh * group + (blockIdx.y % parts) * kTileHeads, heads = min(kTileHeads, (kvh + 1) * group - head0);
    const int t0 = blockIdx.x * TQ, t_end = min(tokens, t0 + TQ);
    auto row_token = [&](int row) { return t0 + row / kTileHeads; };
    auto row_head = [&](int row) { return head0 + row % kTileHeads; };
    auto row_used = [&](int row) { return row_token(row) < t_end && row % kTileHeads < heads; };
    for (int i = threadIdx.x; i < NW * NR * width; i += THREADS) {
        const int row = i / width, d = i - row * width;
        qs[i] = d < hd && row_used(row) ? to_f32(q[static_cast<size_t>(row_token(row)) * q_stride + static_cast<size_t>(row_head(row)) * hd + d]) : 0.f;
    }
    if (CTAS > 1) cluster_wait();                       // the others have begun: their shared memory may be written
    for (int a = t0; a < t_end;) {                      // a run of rows of one request
        auto request = [&](int t) { return request_of(seq_of_token[t], positions[t], table_rows, table_width, page_size, status); };
        const int seq = request(a);
        int b = a + 1, low = positions[a], high = low;
        while (b < t_end && request(b) == seq) {
            low = min(low, positions[b]);
            high = max(high, positions[b]);
            ++b;
        }
        if (seq < 0) {                                  // padded tokens of a fixed-size batch
            for (int row = warp; rank == 0 && row < TQ * kTileHeads; row += NW)
                if (row_used(row) && row_token(row) >= a && row_token(row) < b)
                    for (int d = lane; d < hd; d += 32) out[(static_cast<size_t>(row_token(row)) * nq + row_head(row)) * hd + d] = from_f32<T>(0.f);
            a = b;
            continue;
        }
        const int32_t* table = block_table + static_cast<size_t>(seq) * table_width;
        const int lowest = window > 0 ? max(0, low - window + 1) : 0;
        int pos[NR];
        float M[NR], L[NR], A[NR][G], m[NR], l[NR], acc[NR][G];         // (capitals: the streams before, where the CTA has all)
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = warp * NR + r;
            pos[r] = row_used(row) && row_token(row) >= a && row_token(row) < b ? positions[row_token(row)] : -1;      // -1: not of this run
            M[r] = -INFINITY;
            L[r] = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) A[r][j] = 0.f;
        }
        int begin = 0;                                  // the stream's first key
        uint32_t kw[KW], kp[KW], vh[VW], vp[VW];
        // `index` counts the stream's keys; find: the rows of the THREADS keys from those on
        auto key_of = [&](int index) { return stream_key(begin, index); };
        auto find = [&](int index, int buf) {
            const int key = key_of(index + threadIdx.x);
            size_t at = ~size_t(0);
            if (key >= lowest && key <= high) {
                const int index = key / page_size, page = index < table_width ? table[index] : -1;
                if (page < 0 || page >= num_pages)
                    four::complain(status, four::kCodeNoPage);
                else
                    at = ((static_cast<size_t>(page) * nkv + kvh) * page_size + key % page_size) * bytes;
            }
            row_at[buf][threadIdx.x] = at;
        };
        auto rows_of = [&](int index) { return row_at[index / THREADS & 1] + index % THREADS; };
        auto fetch = [&](const size_t* rows) {          // words of keys: 4 G a row; half words of values: 8 G
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const int w = threadIdx.x + i * THREADS, j = w / (4 * G);
                if (w >= 32 * 4 * G || rows[j] == ~size_t(0)) continue;
                const uint32_t* row = reinterpret_cast<const uint32_t*>(k_pages + rows[j]);
                kw[i] = row[w % (4 * G)];
                kp[i] = row[4 * G + w % G];
            }
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const int w = threadIdx.x + i * THREADS, j = w / (8 * G);
                if (w >= 32 * 8 * G || rows[j] == ~size_t(0)) continue;
                const uint8_t* row = v_pages + rows[j];
                vh[i] = reinterpret_cast<const uint16_t*>(row)[w % (8 * G)];
                vp[i] = reinterpret_cast<const uint32_t*>(row + 16 * G)[w % G];
            }
        };
        auto spread = [&](const size_t* rows) {         // as the numbers they stand for; zeros for a key without a row
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const int w = threadIdx.x + i * THREADS, j = w / (4 * G), in = w % (4 * G);
                if (w >= 32 * 4 * G) continue;
                const bool there = rows[j] != ~size_t(0);
                const float s = there ? four::bf16_low(kp[i]) : 0.f, c = there ? four::bf16_high(kp[i]) : 0.f;
                float* to = ks + j * kld + 32 * (in % G) + 8 * (in / G);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float4*>(to + 4 * h) =
                        make_float4(four::value_of(kw[i] >> (16 * h) & 15u, s, c), four::value_of(kw[i] >> (16 * h + 4) & 15u, s, c),
                                    four::value_of(kw[i] >> (16 * h + 8) & 15u, s, c), four::value_of(kw[i] >> (16 * h + 12) & 15u, s, c));
            }
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const int w = threadIdx.x + i * THREADS, j = w / (8 * G), in = w % (8 * G);
                if (w >= 32 * 8 * G) continue;
                const bool there = rows[j] != ~size_t(0);
                const float s = there ? four::bf16_low(vp[i]) : 0.f, c = there ? four::bf16_high(vp[i]) : 0.f;
                *reinterpret_cast<float4*>(vs + j * width + 32 * (in % G) + 4 * (in / G)) =
                    make_float4(four::value_of(vh[i] & 15u, s, c), four::value_of(vh[i] >> 4 & 15u, s, c), four::value_of(vh[i] >> 8 & 15u, s, c),
                                four::value_of(vh[i] >> 12, s, c));
            }
        };
        for (int stream = rank; stream < kStreams; stream += CTAS) {
            begin = stream_begin(lowest, stream);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                m[r] = -INFINITY;
                l[r] = 0.f;
#pragma unroll
                for (int j = 0; j < G; ++j) acc[r][j] = 0.f;
            }
            if (begin > high) continue;                 // (for the whole CTA)
            __syncthreads();                                // the queries are there, the run before has left the tiles
            find(0, 0);
            if (key_of(THREADS) <= high) find(THREADS, 1);
            __syncthreads();
            if (begin <= high) fetch(rows_of(0));
            for (int index = 0; key_of(index) <= high; index += 32) {
                const int base = key_of(index);
                // (the rows before this THREADS keys' have been read by all)
                if (index && index % THREADS == 0 && key_of(index + THREADS) <= high) find(index + THREADS, (index / THREADS + 1) & 1);
                spread(rows_of(index));
                __syncthreads();
                const bool there = rows_of(index)[lane] != ~size_t(0);
                if (key_of(index + 32) <= high) fetch(rows_of(index + 32));
                const int key = base + lane;
                const float* k_row = ks + lane * kld;
                float s[NR];
                unsigned valid[NR], any = 0;
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const int first = window > 0 ? max(0, pos[r] - window + 1) : 0;
                    valid[r] = __ballot_sync(0xffffffffu, there && key >= first && key <= pos[r]);
                    any |= valid[r];
                    s[r] = 0.f;
                }
                if (any) {
                    const float* q_row = qs + warp * NR * width;
#pragma unroll
                    for (int d = 0; d < width; d += 4) {
                        const float4 kv = *reinterpret_cast<const float4*>(k_row + d);
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            const float4 qv = *reinterpret_cast<const float4*>(q_row + r * width + d);
                            s[r] = fmaf(qv.x, kv.x, s[r]);
                            s[r] = fmaf(qv.y, kv.y, s[r]);
                            s[r] = fmaf(qv.z, kv.z, s[r]);
                            s[r] = fmaf(qv.w, kv.w, s[r]);
                        }
                    }
                    float p[NR];
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        p[r] = 0.f;
                        if (!valid[r]) continue;
                        const bool ok = (valid[r] >> lane) & 1u;
                        float z = s[r] * scale;
                        if (softcap > 0.f) z = softcap * tanhf(z / softcap);
                        if (slopes) z = __fadd_rn(z, -__fmul_rn(slopes[row_head(warp * NR + r)], static_cast<float>(pos[r] - key)));
                        z = ok ? z : -INFINITY;
                        const float m_new = fmaxf(m[r], warp_max(z));
                        p[r] = ok ? expf(z - m_new) : 0.f;
                        const float corr = expf(m[r] - m_new);
                        l[r] = l[r] * corr + warp_sum(p[r]);
#pragma unroll
                        for (int j = 0; j < G; ++j) acc[r][j] *= corr;
                        m[r] = m_new;
                    }
                    // a weight of 0 adds nothing: its key's values are numbers, or zeros
                    __syncwarp();
#pragma unroll
                    for (int r = 0; r < NR; ++r) reinterpret_cast<float*>(weights[warp * NR + r])[lane] = p[r];
                    __syncwarp();
                    const int last = 31 - __clz(any);
                    for (int j4 = (__ffs(any) - 1) / 4; j4 <= last / 4; ++j4) {
                        float4 w[NR];
#pragma unroll
                        for (int r = 0; r < NR; ++r) w[r] = weights[warp * NR + r][j4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int j = 0; j < G; ++j)
                                {
                                    const float v = vs[(4 * j4 + e) * width + 32 * j + lane];
#pragma unroll
                                    for (int r = 0; r < NR; ++r) acc[r][j] = fmaf((&w[r].x)[e], v, acc[r][j]);
                                }
                    }
                }
                __syncthreads();                            // the tiles have been read
            }
            if (CTAS == 1)
#pragma unroll
                for (int r = 0; r < NR; ++r) join(M[r], L[r], A[r], m[r], l[r], acc[r]);
        }
        auto finish = [&](int row, float M, float L, float(&A)[G]) {
            if (sinks) {
                const float sink = sinks[row_head(row)], m_new = fmaxf(M, sink), corr = expf(M - m_new);
                L = L * corr + expf(sink - m_new);
#pragma unroll
                for (int j = 0; j < G; ++j) A[j] *= corr;
            }
            const float inv = L == 0.f ? 0.f : 1.f / L;
            T* out_row = out + (static_cast<size_t>(row_token(row)) * nq + row_head(row)) * hd;
#pragma unroll
            for (int j = 0; j < G; ++j)
                if (32 * j + lane < hd) out_row[32 * j + lane] = from_f32<T>(A[j] * inv);
        };
        if constexpr (CTAS == 1) {
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if (pos[r] >= 0) finish(warp * NR + r, M[r], L[r], A[r]);
        } else {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int row = warp * NR + r;
                float* to = joined[rank][row / kStreams];
                const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to)), owner = row % kStreams;
#pragma unroll
                for (int j = 0; j < G; ++j) store_cluster(at + 4 * (32 * j + lane), owner, acc[r][j]);
                if (lane < 2) store_cluster(at + 4 * (32 * G + lane), owner, lane ? l[r] : m[r]);
            }
            cluster_arrive();
            cluster_wait();
            for (int own = warp; own < OWN; own += NW) {
                const int row = own * kStreams + rank;
                if (row >= NW * NR || !row_used(row) || row_token(row) < a || row_token(row) >= b) continue;
                float M = -INFINITY, L = 0.f, A[G];
#pragma unroll
                for (int j = 0; j < G; ++j) A[j] = 0.f;
                for (int from = 0; from < kStreams; ++from) {
                    float part[G];
#pragma unroll
                    for (int j = 0; j < G; ++j) part[j] = joined[from][own][32 * j + lane];
                    join(M, L, A, joined[from][own][32 * G], joined[from][own][32 * G + 1], part);
                }
                finish(row, M, L, A);
            }
            if (b < t_end) {            // the next run's streams come to the same places
                cluster_arrive();
                cluster_wait();
            }
        }
        a = b;
    }
}

}  // namespace stride

using namespace stride;

struct Int4Attention {
    const void* q;                  // [tokens, q_stride] with head h at columns [h hd, (h + 1) hd)
    void* out;                      // [tokens, nq hd]
    const uint8_t* k_pages;         // [num_pages, nkv, page_size, 20 ceil(hd / 32)]
    const uint8_t* v_pages;
    const int32_t* block_table;     // [requests, table_width]
    const int32_t* seq_of_token;
    const int32_t* positions;
    const float* sinks;
    const float* slopes;
    int* status;
    cudaStream_t stream;
    int q_stride, num_pages, table_width, tokens, nq, nkv, hd, page_size, window;
    float scale, softcap;
    int dtype, neighbours;          // neighbours: rows next to each other are mostly of one request (only the time depends on it)
    int table_rows, bound;          // bound: about how many keys a row has at the most (only the time depends on it)
};

static_assert(sizeof(Int4Attention) == 152, "the record that the caller packs");

template <typename T, int G, int TQ, int NW, int NR, int CTAS>
static int launch_tiles(const Int4Attention& a) {
    constexpr int width = 32 * G, bytes = (32 * (width + 4) + 32 * width + NW * NR * width) * 4;
    const auto kernel = attention_int4_tile_kernel<T, G, TQ, NW, NR, CTAS>;
    const cudaError_t e = allow_shared<attention_int4_tile_kernel<T, G, TQ, NW, NR, CTAS>>(bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int group = a.nq / a.nkv, ctas_y = a.nkv * ((group + kTileHeads - 1) / kTileHeads);
    if (ctas_y > 65535) return STRIDE_UNSUPPORTED;
    stride::launch_clusters(kernel, dim3((a.tokens + TQ - 1) / TQ, ctas_y, CTAS), dim3(NW * 32), bytes, a.stream, CTAS, static_cast<const T*>(a.q), a.q_stride,
                   static_cast<T*>(a.out), a.k_pages, a.v_pages, a.num_pages, a.block_table, a.table_rows, a.table_width, a.seq_of_token, a.positions, a.tokens, a.nq,
                   a.nkv, a.hd, a.page_size, a.scale, a.window, a.softcap, a.sinks, a.slopes, a.status);
    return STRIDE_LAUNCH_STATUS();
}

template <typename T, int G>
static int launch_tiles_of(const Int4Attention& a) {
    // Eight CTAs cut the chain of a row's keys to an eighth and cost their starts and a join, so they pay where there are more keys than CTAs to run
    // side by side. Measured, one CTA against eight, us: 2 x 50 rows at 1000 keys (100 CTAs) 103 / 38; 8 single rows at 2000 (64) 181 / 47; 1 at
    // 8000 (8) 707 / 110; 64 at 4000 (512) 521 / 430; but 64 at 500 (512) 75 / 85, 512 rows in a prompt (512) 77 / 93, 8 x 100 at 700 (1600)
    // 364 / 501, 2048 in a prompt (4096) 2793 / 3175, 16 rows of 20 keys (16) 4.8 / 6.2.
    const int tile = a.neighbours ? 4 : 1;
    const long long keys = a.window > 0 ? min(a.window, a.bound) : a.bound;
    const long long ctas = static_cast<long long>((a.tokens + tile - 1) / tile) * a.nkv * ((a.nq / a.nkv + kTileHeads - 1) / kTileHeads);
    if (keys > 4 * kStretch && keys > ctas) return a.neighbours ? launch_tiles<T, G, 4, 8, 2, kStreams>(a) : launch_tiles<T, G, 1, 4, 1, kStreams>(a);
    // Eight rows a CTA, four to a warp, where that still leaves four CTAs an SM: a key read from shared memory meets twice the rows (2048 rows in a
    // prompt 2794 / 2276 us, 8 x 100 at 700 364 / 359, but 32 x 16 at 200 with 512 CTAs 35 / 41).
    if constexpr (G <= 4)           // (the registers' sake)
        if (a.neighbours && ctas >= 8 * 148) return launch_tiles<T, G, 8, 8, 4, 1>(a);
    return a.neighbours ? launch_tiles<T, G, 4, 8, 2, 1>(a) : launch_tiles<T, G, 1, 4, 1, 1>(a);
}

template <typename T>
static int launch_exact(const Int4Attention& a) {
    switch (four::groups_of(a.hd)) {
        case 1: return launch_tiles_of<T, 1>(a);
        case 2: return launch_tiles_of<T, 2>(a);
        case 3: return launch_tiles_of<T, 3>(a);
        case 4: return launch_tiles_of<T, 4>(a);
        case 5: return launch_tiles_of<T, 5>(a);
        case 6: return launch_tiles_of<T, 6>(a);
        case 7: return launch_tiles_of<T, 7>(a);
        case 8: return launch_tiles_of<T, 8>(a);
    }
    return STRIDE_UNSUPPORTED;
}

// A key whose page is none of the cache's is left out, and the status word says so.
extern "C" int stride_attention_int4_exact(const void* record) {
    const Int4Attention a = read_record<Int4Attention>(record);
    if (a.tokens < 0 || a.nq <= 0 || a.nkv <= 0 || a.hd <= 0 || a.page_size <= 0 || a.table_width <= 0 || a.table_rows <= 0 || a.num_pages <= 0 || a.window < 0 ||
        a.softcap < 0.f || a.nq % a.nkv)
        return STRIDE_BAD_ARGUMENT;
    if (a.hd > four::kMaxHeadDim || (reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) % 4) return STRIDE_UNSUPPORTED;
    if (a.tokens == 0) return 0;
    if (a.dtype == STRIDE_DTYPE_F32) return launch_exact<float>(a);
    return a.dtype == STRIDE_DTYPE_BF16 ? launch_exact<__nv_bfloat16>(a) : STRIDE_BAD_ARGUMENT;
}
