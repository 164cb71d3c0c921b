// Attention over a paged cache held in 4 bits (int4_cache.cuh): the exact kernel.
//
// The rule is that of attention_generic.cu, the numbers are those the rows stand for: softmax(q k^T scale) v over the keys j <= p (and
// j > p - window), scores capped at c tanh(s / c), a penalty slope_h (p - j), a sink per head in the denominator. One warp owns one (token,
// query head); keys are walked in groups of 32 aligned to position 0 with an online softmax in 32 bits, so the order of every sum
// depends on p alone: a token's result has the same bits in a whole prompt, in a portion or alone, on whatever pages.
#include "int4_cache.cuh"

namespace stride {

constexpr int kExactWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kExactWarps * 32)
attention_int4_exact_kernel(const T* __restrict__ q, int q_stride, T* __restrict__ out, const uint8_t* __restrict__ k_pages,
                            const uint8_t* __restrict__ v_pages, int num_pages, const int32_t* __restrict__ block_table, int table_width,
                            const int32_t* __restrict__ seq_of_token, const int32_t* __restrict__ positions, int nq, int nkv, int hd, int page_size,
                            float scale, int window, float softcap, const float* __restrict__ sinks, const float* __restrict__ slopes, int* status) {
    pdl_trigger();
    pdl_wait();
    __shared__ float q_smem[kExactWarps][four::kMaxHeadDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = blockIdx.x, head = blockIdx.y * kExactWarps + warp;
    if (head >= nq) return;
    const int G = four::groups_of(hd), bytes = four::row_bytes(hd);
    T* out_row = out + (static_cast<size_t>(t) * nq + head) * hd;
    const int seq = seq_of_token[t];
    if (seq < 0) {      // a padded token of a fixed-size batch
        for (int d = lane; d < hd; d += 32) out_row[d] = from_f32<T>(0.f);
        return;
    }
    const int pos = positions[t], kvh = head / (nq / nkv);
    const int first = window > 0 ? max(0, pos - window + 1) : 0;
    const int32_t* table = block_table + static_cast<size_t>(seq) * table_width;
    float* qs = q_smem[warp];
    const T* q_row = q + static_cast<size_t>(t) * q_stride + static_cast<size_t>(head) * hd;
    for (int d = lane; d < 32 * G; d += 32) qs[d] = d < hd ? to_f32(q_row[d]) : 0.f;
    __syncwarp();

    const float slope = slopes ? slopes[head] : 0.f;
    float m = -INFINITY, l = 0.f, acc[four::kMaxGroups];
#pragma unroll
    for (int j = 0; j < four::kMaxGroups; ++j) acc[j] = 0.f;
    for (int base = first / 32 * 32; base <= pos; base += 32) {
        const int key = base + lane;
        bool ok = key >= first && key <= pos;
        size_t row = 0;
        if (ok) {
            const int index = key / page_size, page = index < table_width ? table[index] : -1;
            if (page < 0 || page >= num_pages) {
                four::complain(status, four::kCodeNoPage);
                ok = false;
            } else {
                row = ((static_cast<size_t>(page) * nkv + kvh) * page_size + key % page_size) * bytes;
            }
        }
        float s = -INFINITY;
        if (ok) {
            const uint32_t* words = reinterpret_cast<const uint32_t*>(k_pages + row);
            float dot = 0.f;
            for (int g = 0; g < G; ++g) {
                const uint32_t p = words[4 * G + g];
                const float gs = four::bf16_low(p), gc = four::bf16_high(p);
                for (int a = 0; a < 4; ++a) {
                    const uint32_t w = words[a * G + g];
#pragma unroll
                    for (int i = 0; i < 8; ++i) dot = fmaf(qs[32 * g + 8 * a + i], four::value_of(w >> (4 * i) & 15u, gs, gc), dot);
                }
            }
            s = dot * scale;
            if (softcap > 0.f) s = softcap * tanhf(s / softcap);
            if (slopes) s = __fadd_rn(s, -__fmul_rn(slope, static_cast<float>(pos - key)));
        }
        unsigned valid = __ballot_sync(0xffffffffu, ok);
        if (!valid) continue;
        const float m_new = fmaxf(m, warp_max(s));
        const float p = ok ? expf(s - m_new) : 0.f;
        const float corr = expf(m - m_new);
        l = l * corr + warp_sum(p);
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j) acc[j] *= corr;
        for (; valid; valid &= valid - 1) {
            const int from = __ffs(valid) - 1;
            const float pj = __shfl_sync(0xffffffffu, p, from);
            const uint8_t* v_row = v_pages + __shfl_sync(0xffffffffu, row, from);
#pragma unroll
            for (int j = 0; j < four::kMaxGroups; ++j)
                if (j < G) {
                    const uint32_t n = static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(v_row)[(lane >> 2) * G + j]) >> (4 * (lane & 3)) & 15u;
                    const uint32_t params = reinterpret_cast<const uint32_t*>(v_row + 16 * G)[j];
                    acc[j] = fmaf(pj, four::value_of(n, four::bf16_low(params), four::bf16_high(params)), acc[j]);
                }
        }
        m = m_new;
    }
    if (sinks) {
        const float sink = sinks[head], m_new = fmaxf(m, sink), corr = expf(m - m_new);
        l = l * corr + expf(sink - m_new);
#pragma unroll
        for (int j = 0; j < four::kMaxGroups; ++j) acc[j] *= corr;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;         // 0: no key had a page
#pragma unroll
    for (int j = 0; j < four::kMaxGroups; ++j)
        if (32 * j + lane < hd) out_row[32 * j + lane] = from_f32<T>(acc[j] * inv);
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
    int dtype;
};

static_assert(sizeof(Int4Attention) == 136, "the record that the caller packs");

// A key whose page is none of the cache's is left out, and the status word says so.
extern "C" int stride_attention_int4_exact(const void* record) {
    const Int4Attention a = read_record<Int4Attention>(record);
    if (a.tokens < 0 || a.nq <= 0 || a.nkv <= 0 || a.hd <= 0 || a.page_size <= 0 || a.table_width <= 0 || a.num_pages <= 0 || a.window < 0 ||
        a.softcap < 0.f || a.nq % a.nkv)
        return STRIDE_BAD_ARGUMENT;
    const int ctas_y = (a.nq + kExactWarps - 1) / kExactWarps;
    if (a.hd > four::kMaxHeadDim || ctas_y > 65535 || (reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) % 4)
        return STRIDE_UNSUPPORTED;
    if (a.tokens == 0) return 0;
    const dim3 grid(a.tokens, ctas_y), block(kExactWarps * 32);
    if (a.dtype == STRIDE_DTYPE_F32)
        stride::launch(attention_int4_exact_kernel<float>, grid, block, 0, a.stream, static_cast<const float*>(a.q), a.q_stride,
                       static_cast<float*>(a.out), a.k_pages, a.v_pages, a.num_pages, a.block_table, a.table_width, a.seq_of_token, a.positions, a.nq,
                       a.nkv, a.hd, a.page_size, a.scale, a.window, a.softcap, a.sinks, a.slopes, a.status);
    else if (a.dtype == STRIDE_DTYPE_BF16)
        stride::launch(attention_int4_exact_kernel<__nv_bfloat16>, grid, block, 0, a.stream, static_cast<const __nv_bfloat16*>(a.q), a.q_stride,
                       static_cast<__nv_bfloat16*>(a.out), a.k_pages, a.v_pages, a.num_pages, a.block_table, a.table_width, a.seq_of_token, a.positions,
                       a.nq, a.nkv, a.hd, a.page_size, a.scale, a.window, a.softcap, a.sinks, a.slopes, a.status);
    else
        return STRIDE_BAD_ARGUMENT;
    return STRIDE_LAUNCH_STATUS();
}
