// Copies of pages inside the pools of a cache: for each pair (from, to) page `to` of every pool and layer becomes page `from`.
//
// A pool is [layers, num_pages, page_bytes]. The pairs travel as the kernel's parameters, so a call needs neither a copy to the device nor
// memory of its own, and a captured graph holds the pairs it was captured with. No page is both read and written, so the order of the
// copies does not matter (the caller checks). Attention may ask for keys of earlier steps before the kernel in front of it has ended: this one
// lets nothing start early. Bound by the bytes: every page is read once and written once. 512 pages of 10 KB for
// keys and values in 32 layers are 671 MB in 105 us, 0.98 of the copy rate; 8 pages of 32 KB (34 MB) 5.5 us, out of L2.
// A thread has kCopyPacks packs of 16 bytes under way; smaller packs serve pages whose size or address is odd.
#include "common.cuh"

namespace stride {

constexpr int kCopyThreads = 256;
constexpr int kCopyPools = 8;
constexpr int kCopyPairs = 448;         // what fits into 4 KB of parameters beside the pools
constexpr int kCopyPacks = 4;           // packs a thread has under way at once

struct PageCopies {
    unsigned char* base[kCopyPools];
    long long page_bytes[kCopyPools], layer_bytes[kCopyPools];
    int layers[kCopyPools];
    int2 pairs[kCopyPairs];
};

// CTA (x, y, z): part x of the page, pair y, layer z counted over all pools. P: the pack that bases and page sizes are multiples of.
template <typename P>
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ PageCopies a) {
    int layer = blockIdx.z, pool = 0;
    while (layer >= a.layers[pool]) layer -= a.layers[pool++];
    const long long packs = a.page_bytes[pool] / static_cast<long long>(sizeof(P));
    const long long first = static_cast<long long>(blockIdx.x) * kCopyThreads * kCopyPacks + threadIdx.x;
    const int2 pair = a.pairs[blockIdx.y];
    unsigned char* base = a.base[pool] + layer * a.layer_bytes[pool];
    const P* from = reinterpret_cast<const P*>(base + pair.x * a.page_bytes[pool]);
    P* to = reinterpret_cast<P*>(base + pair.y * a.page_bytes[pool]);
    P v[kCopyPacks];
#pragma unroll
    for (int i = 0; i < kCopyPacks; ++i)
        if (first + i * kCopyThreads < packs) v[i] = from[first + i * kCopyThreads];
#pragma unroll
    for (int i = 0; i < kCopyPacks; ++i)
        if (first + i * kCopyThreads < packs) to[first + i * kCopyThreads] = v[i];
}

template <typename P>
void launch_copies(const PageCopies& a, long long most_bytes, int pairs, int layers, cudaStream_t stream) {
    const long long packs = most_bytes / static_cast<long long>(sizeof(P)), per_cta = kCopyThreads * kCopyPacks;
    stride::launch_alone(page_copy_kernel<P>, dim3(static_cast<unsigned>((packs + per_cta - 1) / per_cta), pairs, layers), dim3(kCopyThreads), 0, stream, a);
}

}  // namespace stride

using namespace stride;

// pools: of each of the n_pools pools its device address, layers, pages and bytes of a page. from, to: `pairs` page numbers of every pool. All of
// them host memory. The caller has checked that no page of `to` comes twice or also in `from`.
extern "C" int stride_copy_pages(const long long* pools, int n_pools, const int* from, const int* to, int pairs, cudaStream_t stream) {
    if (n_pools < 0 || pairs < 0) return STRIDE_BAD_ARGUMENT;
    for (int p = 0; p < n_pools; ++p) {
        const long long* q = pools + 4 * p;
        if (q[0] == 0 || q[1] <= 0 || q[2] <= 0 || q[3] <= 0) return STRIDE_BAD_ARGUMENT;
        if (q[1] > 65535 || q[3] > (1LL << 40)) return STRIDE_UNSUPPORTED;
        for (int i = 0; i < pairs; ++i)
            if (from[i] < 0 || to[i] < 0 || from[i] >= q[2] || to[i] >= q[2]) return STRIDE_BAD_ARGUMENT;
    }
    for (int p0 = 0; p0 < n_pools;) {
        PageCopies a;
        long long all = 0, most = 0;
        int layers = 0, n = 0;                  // a launch takes up to eight pools and 65535 layers
        for (; n < kCopyPools && p0 + n < n_pools && layers + pools[4 * (p0 + n) + 1] <= 65535; ++n) {
            const long long* q = pools + 4 * (p0 + n);
            a.base[n] = reinterpret_cast<unsigned char*>(q[0]);
            a.layers[n] = static_cast<int>(q[1]);
            a.page_bytes[n] = q[3];
            a.layer_bytes[n] = q[3] * q[2];
            layers += a.layers[n];
            all |= q[0] | q[3];
            most = most > q[3] ? most : q[3];
        }
        p0 += n;
        for (int i0 = 0; i0 < pairs; i0 += kCopyPairs) {
            const int count = pairs - i0 < kCopyPairs ? pairs - i0 : kCopyPairs;
            for (int i = 0; i < count; ++i) a.pairs[i] = make_int2(from[i0 + i], to[i0 + i]);
            if (all % 16 == 0)
                launch_copies<uint4>(a, most, count, layers, stream);
            else if (all % 4 == 0)
                launch_copies<uint32_t>(a, most, count, layers, stream);
            else
                launch_copies<uint8_t>(a, most, count, layers, stream);
            const int code = STRIDE_LAUNCH_STATUS();
            if (code) return code;
        }
    }
    return 0;
}
