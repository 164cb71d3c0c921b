// What stands between the q/k/v projection and attention, in one pass: bias, an RMS norm with a weight on every query and key head, the
// rotation, and the write of keys and values into their pages, as they are or held in 4 bits (int4_cache.cuh).
//   x = row + bias;  y = x rsqrt(mean(x^2) + eps) w (queries and keys, where weights are given);  entry i turns with entry i + hd/2
// Everything is 32-bit between the load and the store: a query, key or value is rounded once, to the element type or to 4 bits.
//
// Every row is read and written once, and nothing is reduced over more than a head, so the bytes are the floor: 2048 tokens of 32 + 8 heads of 128
// in bfloat16 move 51 MB, 7.9 us; the launch takes 11.4 us. Its loads come from L2 or memory with a single item in flight a lane group, so warps
// wait for them, and instructions issue in 60 % of the cycles. In 4 bits the same tokens with norms and a bias take 14.5 us: the extra time
// is the search of each group's extremes and the rounding. A step of 64 tokens takes 2.3 us, a launch's latency.
#include "int4_cache.cuh"

namespace stride {

constexpr int kWriteWarps = 4;

struct HeadWrite {                  // a record that the caller packs: addresses, then 64-bit, then 32-bit numbers
    const void* rows;               // [tokens, (nq + 2 nkv) hd]
    void* q_out;                    // head h of token t at q_out[t * q_out_stride + h * hd]
    const float* bias;              // [(nq + 2 nkv) hd] or null
    const float* q_norm;            // [hd], both or none
    const float* k_norm;
    const int32_t* positions;
    const int32_t* slots;           // null: nothing is stored
    const float* cos;               // [num_positions, hd / 2]
    const float* sin;
    void* k_pages;
    void* v_pages;
    int* status;
    cudaStream_t stream;
    long long q_out_stride;
    int num_positions, num_pages, bits4, tokens, nq, nkv, hd, page_size, rotate, dtype;
    float eps;
};

static_assert(sizeof(HeadWrite) == 160, "the record that the caller packs");

// A warp a unit: a query head, or a key head with its value head. Lane l holds entry 32 j + l of the head in x[j], so a group of 32 is
// one register of the warp. The form for every even head size: its loads are 2 or 4 bytes a lane, and where the one below can run it takes three
// times as long (a prompt of 2048 tokens 42 us for 11, in 4 bits 81 with the read back for 22); 333 tokens of 32 bits with heads of 96 take 4.3.
template <typename T, bool FOUR>
__global__ void __launch_bounds__(kWriteWarps * 32) head_write_kernel(const HeadWrite a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float staged[kWriteWarps][four::kMaxHeadDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x, unit = blockIdx.y * kWriteWarps + warp;
    if (unit >= a.nq + a.nkv) return;
    const int hd = a.hd, half = hd >> 1, G = four::groups_of(hd), heads = a.nq + 2 * a.nkv;
    const T* row = static_cast<const T*>(a.rows) + static_cast<size_t>(t) * heads * hd;
    const int pos = a.rotate ? a.positions[t] : 0;
    if (a.rotate && (pos < 0 || pos >= a.num_positions)) {
        if (lane == 0) four::complain(a.status, four::kCodeNoPosition);
        return;
    }
    const bool is_q = unit < a.nq;
    const int slot = a.slots != nullptr && !is_q ? a.slots[t] : -1;
    if (!is_q && slot < 0) return;
    const int page = is_q ? 0 : slot / a.page_size, offset = is_q ? 0 : slot % a.page_size;
    if (page >= a.num_pages) {
        if (lane == 0) four::complain(a.status, four::kCodeNoSlot);
        return;
    }
    const int kvh = unit - a.nq;
    float x[four::kMaxGroups], v[four::kMaxGroups];
    auto load = [&](int head, float* out) {
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j) {
            const int d = 32 * j + lane;
            out[j] = 0.f;
            if (j < G && d < hd) {
                out[j] = to_f32(row[static_cast<size_t>(head) * hd + d]);
                if (a.bias != nullptr) out[j] = __fadd_rn(out[j], a.bias[static_cast<size_t>(head) * hd + d]);
            }
        }
    };
    load(unit, x);                                             // key head kvh is head nq + kvh of the row
    if (!is_q) load(unit + a.nkv, v);
    const float* weight = is_q ? a.q_norm : a.k_norm;
    if (weight != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j) sum = fmaf(x[j], x[j], sum);
        const float inv = rsqrtf(__fadd_rn(__fdiv_rn(warp_sum(sum), static_cast<float>(hd)), a.eps));
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j)
            if (32 * j + lane < hd) x[j] = __fmul_rn(__fmul_rn(x[j], inv), weight[32 * j + lane]);
    }
    if (a.rotate) {
        const float* cs = a.cos + static_cast<size_t>(pos) * half;
        const float* sn = a.sin + static_cast<size_t>(pos) * half;
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j)
            if (32 * j + lane < hd) staged[warp][32 * j + lane] = x[j];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j) {
            const int d = 32 * j + lane;
            if (d < half)
                x[j] = __fadd_rn(__fmul_rn(x[j], cs[d]), __fmul_rn(-staged[warp][d + half], sn[d]));
            else if (d < hd)
                x[j] = __fadd_rn(__fmul_rn(x[j], cs[d - half]), __fmul_rn(staged[warp][d - half], sn[d - half]));
        }
    }
    if (is_q) {
        T* out = static_cast<T*>(a.q_out) + static_cast<size_t>(t) * a.q_out_stride + static_cast<size_t>(unit) * hd;
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j)
            if (32 * j + lane < hd) out[32 * j + lane] = from_f32<T>(x[j]);
        return;
    }
    const size_t at = (static_cast<size_t>(page) * a.nkv + kvh) * a.page_size + offset;
    if constexpr (!FOUR) {
        T* k = static_cast<T*>(a.k_pages) + at * hd;
        T* w = static_cast<T*>(a.v_pages) + at * hd;
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j)
            if (32 * j + lane < hd) {
                k[32 * j + lane] = from_f32<T>(x[j]);
                w[32 * j + lane] = from_f32<T>(v[j]);
            }
    } else {
        const int bytes = four::row_bytes(hd);
        uint8_t* rows[2] = {static_cast<uint8_t*>(a.k_pages) + at * bytes, static_cast<uint8_t*>(a.v_pages) + at * bytes};
        float s[2][four::kMaxGroups], c[2][four::kMaxGroups];
        bool fine = true;
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int j = 0; j < four::kMaxGroups; ++j) {
                if (j >= G) continue;
                const bool there = 32 * j + lane < hd;
                const float e = which ? v[j] : x[j];
                fine = fine && (!there || fabsf(e) < four::kMaxEntry);
                float lo = there ? e : INFINITY, hi = there ? e : -INFINITY;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                }
                four::group_params(lo, hi, s[which][j], c[which][j]);
            }
        fine = __all_sync(0xffffffffu, fine);
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int j = 0; j < four::kMaxGroups; ++j) {
                if (j >= G) continue;
                const float e = which ? v[j] : x[j];
                float sj = s[which][j], cj = c[which][j];
                uint32_t n = 8;
                if (!fine)
                    sj = cj = which ? 0.f : __int_as_float(0x7fc00000);
                else if (32 * j + lane < hd && sj > 0.f)
                    n = four::number_of(e, cj, __frcp_rn(sj));
                if (which == 0) {
                    uint32_t word = n << (4 * (lane & 7));
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
                    if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(rows[0])[(lane >> 3) * G + j] = word;
                } else {
                    uint32_t word = n << (4 * (lane & 3));
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
                    if ((lane & 3) == 0) reinterpret_cast<uint16_t*>(rows[1])[(lane >> 2) * G + j] = static_cast<uint16_t>(word);
                }
                if (lane == 0) reinterpret_cast<uint32_t*>(rows[which] + 16 * G)[j] = four::pack_params(sj, cj);
            }
    }
}

// The same for head sizes 64, 128 and 256: HD / 8 lanes a head, a lane owns four neighbouring entries of either half, so the pairs that turn
// together meet in one lane, a group of 32 is eight neighbouring lanes, and loads and stores are 8 (bfloat16) or 16 bytes. HD / 8 lanes take
// an item: kQueries query heads of a token, or kPairs of its key heads with their values, whose loads are all under way, beside the position's and
// the slot's, before the first is worked on; angles and weights are read once an item. 2048 tokens of 32 + 8 heads of 128: 21 us with one query
// head an item, 14.3 with two, 11.4 with four, 12.5 with eight; two pairs of keys and values are slower than one, for their registers. CTAs of
// 128 threads, nine an SM: 256 threads, five an SM, take 12.9, 64 threads 12.3.
template <typename T>
struct Four;
template <>
struct Four<float> {
    float4 raw;
    __device__ __forceinline__ void load(const float* p) { raw = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = raw.x; x[1] = raw.y; x[2] = raw.z; x[3] = raw.w; }
    static __device__ __forceinline__ void put(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
};
template <>
struct Four<__nv_bfloat16> {
    uint2 raw;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { raw = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void get(float (&x)[4]) const {
        x[0] = four::bf16_low(raw.x); x[1] = four::bf16_high(raw.x); x[2] = four::bf16_low(raw.y); x[3] = four::bf16_high(raw.y);
    }
    static __device__ __forceinline__ void put(__nv_bfloat16* p, const float (&x)[4]) {
        *reinterpret_cast<uint2*>(p) = make_uint2(four::pack_params(x[0], x[1]), four::pack_params(x[2], x[3]));
    }
};

constexpr int kItemThreads = 128, kQueries = 4, kPairs = 1;

template <typename T, bool FOUR, int HD>
__global__ void __launch_bounds__(kItemThreads, 9) head_write_vec_kernel(const HeadWrite a) {
    constexpr int L = HD / 8, HALF = HD / 2, G = HD / 32;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, i = threadIdx.x % L, heads = a.nq + 2 * a.nkv;
    const uint32_t mask = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << (lane / L * L);       // the lanes of this item
    const uint32_t q_items = (a.nq + kQueries - 1) / kQueries, kv_items = (a.nkv + kPairs - 1) / kPairs;
    uint32_t item = blockIdx.x * (kItemThreads / L) + threadIdx.x / L;             // (the launch sees to it that items fit 31 bits)
    const bool is_q = item < a.tokens * q_items;
    if (!is_q) item -= a.tokens * q_items;
    const int per = is_q ? q_items : kv_items, t = item / static_cast<uint32_t>(per), u0 = item - t * per;      // heads u0, u0 + per, ...
    if (t >= a.tokens) return;
    const T* row = static_cast<const T*>(a.rows) + static_cast<size_t>(t) * heads * HD + 4 * i;
    const int pos = a.rotate ? a.positions[t] : 0;
    const int place = !is_q && a.slots != nullptr ? a.slots[t] : -1;
    float cs[4], sn[4];
    auto angles = [&]() {           // false: there are none for the token's position
        if (!a.rotate) return true;
        if (pos < 0 || pos >= a.num_positions) {
            if (i == 0) four::complain(a.status, four::kCodeNoPosition);
            return false;
        }
        Four<float> c, s;
        c.load(a.cos + static_cast<size_t>(pos) * HALF + 4 * i);
        s.load(a.sin + static_cast<size_t>(pos) * HALF + 4 * i);
        c.get(cs);
        s.get(sn);
        return true;
    };
    auto add_bias = [&](float (&x)[2][4], int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Four<float> add;
            float b[4];
            add.load(a.bias + static_cast<size_t>(u) * HD + h * HALF + 4 * i);
            add.get(b);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[h][e] = __fadd_rn(x[h][e], b[e]);
        }
    };
    float w[2][4];
    auto weights = [&](const float* from) {     // once an item: behind a head's store they would be read again
#pragma unroll
        for (int h = 0; h < 2 && from != nullptr; ++h) {
            Four<float> of;
            of.load(from + h * HALF + 4 * i);
            of.get(w[h]);
        }
    };
    auto norm_and_turn = [&](float (&x)[2][4], bool norm) {
        if (norm) {
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = fmaf(x[h][e], x[h][e], sum);
#pragma unroll
            for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(mask, sum, o);
            const float inv = rsqrtf(__fadd_rn(__fmul_rn(sum, 1.f / HD), a.eps));       // (HD is a power of two: the quotient's bits)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[h][e] = __fmul_rn(__fmul_rn(x[h][e], inv), w[h][e]);
        }
        if (a.rotate) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = x[0][e], q = x[1][e];
                x[0][e] = __fadd_rn(__fmul_rn(p, cs[e]), __fmul_rn(-q, sn[e]));
                x[1][e] = __fadd_rn(__fmul_rn(q, cs[e]), __fmul_rn(p, sn[e]));
            }
        }
    };
    if (is_q) {
        Four<T> in[kQueries][2];
#pragma unroll
        for (int k = 0; k < kQueries; ++k)
            if (u0 + k * per < a.nq) {
                in[k][0].load(row + static_cast<size_t>(u0 + k * per) * HD);
                in[k][1].load(row + static_cast<size_t>(u0 + k * per) * HD + HALF);
            }
        weights(a.q_norm);
        if (!angles()) return;
        T* out = static_cast<T*>(a.q_out) + static_cast<size_t>(t) * a.q_out_stride + 4 * i;
#pragma unroll
        for (int k = 0; k < kQueries; ++k) {
            const int u = u0 + k * per;
            if (u >= a.nq) break;
            float x[2][4];
            in[k][0].get(x[0]);
            in[k][1].get(x[1]);
            if (a.bias != nullptr) add_bias(x, u);
            norm_and_turn(x, a.q_norm != nullptr);
            Four<T>::put(out + static_cast<size_t>(u) * HD, x[0]);
            Four<T>::put(out + static_cast<size_t>(u) * HD + HALF, x[1]);
        }
        return;
    }
    Four<T> in[kPairs][4];
#pragma unroll
    for (int k = 0; k < kPairs; ++k)
        if (u0 + k * per < a.nkv) {
            const T* key = row + static_cast<size_t>(a.nq + u0 + k * per) * HD;
            const T* value = key + static_cast<size_t>(a.nkv) * HD;
            in[k][0].load(key);
            in[k][1].load(key + HALF);
            in[k][2].load(value);
            in[k][3].load(value + HALF);
        }
    weights(a.k_norm);
    if (place < 0 || !angles()) return;
    const int page = place / a.page_size;
    if (page >= a.num_pages) {
        if (i == 0) four::complain(a.status, four::kCodeNoSlot);
        return;
    }
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
        const int u = u0 + k * per;
        if (u >= a.nkv) break;
        float x[2][2][4];                           // key, value
#pragma unroll
        for (int q = 0; q < 4; ++q) in[k][q].get(x[q >> 1][q & 1]);
        if (a.bias != nullptr) {
            add_bias(x[0], a.nq + u);
            add_bias(x[1], a.nq + a.nkv + u);
        }
        norm_and_turn(x[0], a.k_norm != nullptr);
        const size_t at = (static_cast<size_t>(page) * a.nkv + u) * a.page_size + place % a.page_size;
        if constexpr (!FOUR) {
            T* ko = static_cast<T*>(a.k_pages) + at * HD + 4 * i;
            T* vo = static_cast<T*>(a.v_pages) + at * HD + 4 * i;
            Four<T>::put(ko, x[0][0]);
            Four<T>::put(ko + HALF, x[0][1]);
            Four<T>::put(vo, x[1][0]);
            Four<T>::put(vo + HALF, x[1][1]);
        } else {
            float s[2][2], c[2][2];                 // [key, value][half]
            bool fine = true;
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float(&y)[4] = x[w][h];
                    float lo = fminf(fminf(y[0], y[1]), fminf(y[2], y[3])), hi = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
#pragma unroll
                    for (int e = 0; e < 4; ++e) fine = fine && fabsf(y[e]) < four::kMaxEntry;
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) {
                        lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
                        hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
                    }
                    four::group_params(lo, hi, s[w][h], c[w][h]);
                }
            fine = __all_sync(mask, fine);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float(&y)[4] = x[w][h];
                    const int g = h * (G / 2) + i / 8, r = i & 7;              // this lane: entries 4 r .. of group g
                    float sg = s[w][h], cg = c[w][h];
                    uint32_t n = 0x8888u;
                    if (!fine) {
                        sg = cg = w ? 0.f : __int_as_float(0x7fc00000);
                    } else if (sg > 0.f) {
                        const float inverse = __frcp_rn(sg);
                        n = four::number_of(y[0], cg, inverse) | four::number_of(y[1], cg, inverse) << 4 | four::number_of(y[2], cg, inverse) << 8 |
                            four::number_of(y[3], cg, inverse) << 12;
                    }
                    uint8_t* out = static_cast<uint8_t*>(w ? a.v_pages : a.k_pages) + at * (20 * G);
                    // keys: half a word of entries 8 (r / 2) .., values: the 16 bits of entries 4 r ..
                    const int half_word = w ? r * G + g : 2 * ((r >> 1) * G + g) + (r & 1);
                    reinterpret_cast<uint16_t*>(out)[half_word] = static_cast<uint16_t>(n);
                    if (r == 0) reinterpret_cast<uint32_t*>(out + 16 * G)[g] = four::pack_params(sg, cg);
                }
        }
    }
}

template <typename T, bool FOUR, int HD>
void launch_vec(const HeadWrite& a) {
    const long long items = static_cast<long long>(a.tokens) * ((a.nq + kQueries - 1) / kQueries + (a.nkv + kPairs - 1) / kPairs);
    const long long per_cta = kItemThreads / (HD / 8);
    stride::launch(head_write_vec_kernel<T, FOUR, HD>, dim3(static_cast<unsigned>((items + per_cta - 1) / per_cta)), dim3(kItemThreads), 0, a.stream, a);
}
template <typename T, bool FOUR>
bool launch_vec_of(const HeadWrite& a) {        // false: not these sizes, or not aligned
    uintptr_t rows = reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(a.q_out);
    if (!FOUR) rows |= reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages);
    uintptr_t angles = reinterpret_cast<uintptr_t>(a.bias) | reinterpret_cast<uintptr_t>(a.q_norm) | reinterpret_cast<uintptr_t>(a.k_norm);
    if (a.rotate) angles |= reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin);
    if (rows % (4 * sizeof(T)) || angles % 16 || a.q_out_stride % 4 || static_cast<long long>(a.tokens) * (a.nq + a.nkv) > 2147483647LL) return false;
    if (a.hd == 64) launch_vec<T, FOUR, 64>(a);
    else if (a.hd == 128) launch_vec<T, FOUR, 128>(a);
    else if (a.hd == 256) launch_vec<T, FOUR, 256>(a);
    else return false;
    return true;
}

// What the slots of a 4-bit cache stand for: k_out, v_out [n, nkv, hd]. A slot below zero reads as zeros. A warp a row, of any head size.
template <typename T>
__global__ void __launch_bounds__(kWriteWarps * 32)
int4_read_kernel(const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const int32_t* __restrict__ slots, T* __restrict__ k_out,
                 T* __restrict__ v_out, int n, int nkv, int hd, int page_size, int num_pages, int* status) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, G = four::groups_of(hd), bytes = four::row_bytes(hd);
    const long long unit = static_cast<long long>(blockIdx.x) * kWriteWarps + (threadIdx.x >> 5);
    if (unit >= static_cast<long long>(n) * nkv) return;
    const int i = static_cast<int>(unit / nkv), kvh = static_cast<int>(unit % nkv);
    const int slot = slots[i];
    int page = slot < 0 ? -1 : slot / page_size;
    if (page >= num_pages) {
        if (lane == 0) four::complain(status, four::kCodeNoSlot);
        page = -1;
    }
    T* out[2] = {k_out + unit * hd, v_out + unit * hd};
    if (page < 0) {
        for (int d = lane; d < hd; d += 32) out[0][d] = out[1][d] = from_f32<T>(0.f);
        return;
    }
    const size_t at = ((static_cast<size_t>(page) * nkv + kvh) * page_size + slot % page_size) * bytes;
    const uint8_t* rows[2] = {k_pages + at, v_pages + at};
    for (int j = 0; j < G; ++j) {
        const int d = 32 * j + lane;
        if (d >= hd) break;
        const uint32_t kn = reinterpret_cast<const uint32_t*>(rows[0])[(lane >> 3) * G + j] >> (4 * (lane & 7)) & 15u;
        const uint32_t vn = static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(rows[1])[(lane >> 2) * G + j]) >> (4 * (lane & 3)) & 15u;
        const uint32_t kp = reinterpret_cast<const uint32_t*>(rows[0] + 16 * G)[j], vp = reinterpret_cast<const uint32_t*>(rows[1] + 16 * G)[j];
        out[0][d] = from_f32<T>(four::value_of(kn, four::bf16_low(kp), four::bf16_high(kp)));
        out[1][d] = from_f32<T>(four::value_of(vn, four::bf16_low(vp), four::bf16_high(vp)));
    }
}

// The same for head sizes 64, 128 and 256: HD / 8 lanes a row, four neighbouring entries of either half a lane. Bound by the latency of its loads, a slot
// and then 16 and 32 bits at a time out of rows of 80 bytes: 2048 tokens of 8 heads of 128 take 7.5 us for 11 MB, a quarter of the copy rate.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
int4_read_vec_kernel(const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const int32_t* __restrict__ slots, T* __restrict__ k_out,
                     T* __restrict__ v_out, uint32_t units, int nkv, int page_size, int num_pages, int* status) {
    constexpr int L = HD / 8, HALF = HD / 2, G = HD / 32;
    pdl_trigger();
    pdl_wait();
    const int i = threadIdx.x % L, r = i & 7;
    const uint32_t unit = blockIdx.x * (256 / L) + threadIdx.x / L, token = unit / nkv;
    if (unit >= units) return;
    const int slot = slots[token], kvh = unit - token * nkv;
    int page = slot < 0 ? -1 : slot / page_size;
    if (page >= num_pages) {
        if (i == 0) four::complain(status, four::kCodeNoSlot);
        page = -1;
    }
    float y[4][4] = {};
    if (page >= 0) {
        const size_t at = ((static_cast<size_t>(page) * nkv + kvh) * page_size + slot % page_size) * (20 * G);
        uint32_t n[4], p[4];
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t* row = (w ? v_pages : k_pages) + at;
                const int g = h * (G / 2) + i / 8;
                n[2 * w + h] = reinterpret_cast<const uint16_t*>(row)[w ? r * G + g : 2 * ((r >> 1) * G + g) + (r & 1)];
                p[2 * w + h] = reinterpret_cast<const uint32_t*>(row + 16 * G)[g];
            }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[q][e] = four::value_of(n[q] >> (4 * e) & 15u, four::bf16_low(p[q]), four::bf16_high(p[q]));
    }
    const size_t to = static_cast<size_t>(unit) * HD + 4 * i;
    Four<T>::put(k_out + to, y[0]);
    Four<T>::put(k_out + to + HALF, y[1]);
    Four<T>::put(v_out + to, y[2]);
    Four<T>::put(v_out + to + HALF, y[3]);
}

}  // namespace stride

using namespace stride;

// rows: [tokens, (nq + 2 nkv) hd]; q_out: rows of q_out_stride elements (`rows` itself, with its row length, for queries in place).
// bits4: pages hold 4 bits (uint8 [num_pages, nkv, page_size, 20 ceil(hd / 32)]), else elements [num_pages, nkv, page_size, hd]. slots null, or
// a slot below zero: keys and values are not stored. Slots of one launch are distinct. Returns -2 for odd head sizes and those above 256.
extern "C" int stride_head_write(const void* record) {
    const HeadWrite a = read_record<HeadWrite>(record);
    if (a.tokens < 0 || a.nq <= 0 || a.nkv <= 0 || a.hd <= 0 || a.page_size <= 0 || a.num_pages <= 0 ||
        a.q_out_stride < static_cast<long long>(a.nq) * a.hd || (a.q_norm == nullptr) != (a.k_norm == nullptr) || (a.rotate && a.num_positions <= 0) ||
        static_cast<long long>(a.num_pages) * a.page_size > 2147483647LL)
        return STRIDE_BAD_ARGUMENT;
    if (a.hd > four::kMaxHeadDim || (a.rotate && a.hd % 2)) return STRIDE_UNSUPPORTED;
    if (a.bits4 && (reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) % 4) return STRIDE_UNSUPPORTED;
    const int units = a.nq + a.nkv, ctas_y = (units + kWriteWarps - 1) / kWriteWarps;
    if (ctas_y > 65535) return STRIDE_UNSUPPORTED;
    if (a.tokens == 0) return 0;
    if (a.dtype != STRIDE_DTYPE_F32 && a.dtype != STRIDE_DTYPE_BF16) return STRIDE_BAD_ARGUMENT;
    const bool wide = a.dtype == STRIDE_DTYPE_F32;
    if (wide ? (a.bits4 ? launch_vec_of<float, true>(a) : launch_vec_of<float, false>(a))
             : (a.bits4 ? launch_vec_of<__nv_bfloat16, true>(a) : launch_vec_of<__nv_bfloat16, false>(a)))
        return STRIDE_LAUNCH_STATUS();
    const dim3 grid(a.tokens, ctas_y), block(kWriteWarps * 32);
    if (wide)
        a.bits4 ? stride::launch(head_write_kernel<float, true>, grid, block, 0, a.stream, a)
                : stride::launch(head_write_kernel<float, false>, grid, block, 0, a.stream, a);
    else
        a.bits4 ? stride::launch(head_write_kernel<__nv_bfloat16, true>, grid, block, 0, a.stream, a)
                : stride::launch(head_write_kernel<__nv_bfloat16, false>, grid, block, 0, a.stream, a);
    return STRIDE_LAUNCH_STATUS();
}

struct Int4Read {
    const uint8_t* k_pages;
    const uint8_t* v_pages;
    const int32_t* slots;
    void* k_out;            // [n, nkv, hd]
    void* v_out;
    int* status;
    cudaStream_t stream;
    int n, nkv, hd, page_size, num_pages, dtype;
};

static_assert(sizeof(Int4Read) == 80, "the record that the caller packs");

extern "C" int stride_int4_read(const void* record) {
    const Int4Read a = read_record<Int4Read>(record);
    if (a.n < 0 || a.nkv <= 0 || a.hd <= 0 || a.page_size <= 0 || a.num_pages <= 0) return STRIDE_BAD_ARGUMENT;
    if (a.hd > four::kMaxHeadDim || (reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) % 4) return STRIDE_UNSUPPORTED;
    if (a.n == 0) return 0;
    const long long units = static_cast<long long>(a.n) * a.nkv;
    if (a.dtype != STRIDE_DTYPE_F32 && a.dtype != STRIDE_DTYPE_BF16) return STRIDE_BAD_ARGUMENT;
    const bool aligned = (reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)) % 16 == 0;
    if (aligned && (a.hd == 64 || a.hd == 128 || a.hd == 256)) {
        const int rows = 2048 / a.hd;       // of a CTA of 256 threads
        if (units > 2147483647LL) return STRIDE_UNSUPPORTED;
        const dim3 grid(static_cast<unsigned>((units + rows - 1) / rows));
#define STRIDE_READ(T_, HD_)                                                                                                                       \
    stride::launch(int4_read_vec_kernel<T_, HD_>, grid, dim3(256), 0, a.stream, a.k_pages, a.v_pages, a.slots, static_cast<T_*>(a.k_out),           \
                   static_cast<T_*>(a.v_out), static_cast<uint32_t>(units), a.nkv, a.page_size, a.num_pages, a.status)
        if (a.dtype == STRIDE_DTYPE_F32)
            a.hd == 64 ? STRIDE_READ(float, 64) : a.hd == 128 ? STRIDE_READ(float, 128) : STRIDE_READ(float, 256);
        else
            a.hd == 64 ? STRIDE_READ(__nv_bfloat16, 64) : a.hd == 128 ? STRIDE_READ(__nv_bfloat16, 128) : STRIDE_READ(__nv_bfloat16, 256);
#undef STRIDE_READ
        return STRIDE_LAUNCH_STATUS();
    }
    const long long ctas = (static_cast<long long>(a.n) * a.nkv + kWriteWarps - 1) / kWriteWarps;
    if (ctas > 2147483647LL) return STRIDE_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(ctas)), block(kWriteWarps * 32);
    if (a.dtype == STRIDE_DTYPE_F32)
        stride::launch(int4_read_kernel<float>, grid, block, 0, a.stream, a.k_pages, a.v_pages, a.slots, static_cast<float*>(a.k_out),
                       static_cast<float*>(a.v_out), a.n, a.nkv, a.hd, a.page_size, a.num_pages, a.status);
    else
        stride::launch(int4_read_kernel<__nv_bfloat16>, grid, block, 0, a.stream, a.k_pages, a.v_pages, a.slots, static_cast<__nv_bfloat16*>(a.k_out),
                       static_cast<__nv_bfloat16*>(a.v_out), a.n, a.nkv, a.hd, a.page_size, a.num_pages, a.status);
    return STRIDE_LAUNCH_STATUS();
}
