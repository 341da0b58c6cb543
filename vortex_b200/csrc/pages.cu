// Pages copied inside the pools of a cache: a sequence forked (its open page is its own from then on), a cache compacted.
//
// One launch moves up to 2048 pages in up to 64 pools (keys and values of every attention layer hold a page under the same
// number).  The page numbers are host data, the plan being made there; they travel in the launch's parameters: no copy to the
// device that would have to be waited for or kept alive, and a captured launch carries its own.  Each byte is read once and
// written once: memory bounds it (701 pages of 128 KB in ten pools: 280 us, 1.0 of the measured copy bandwidth), launches of a
// page or two the launch itself (one page in ten pools: 1.7 us).
#include <cstdlib>

#include "common.cuh"

namespace vtx {
namespace {

constexpr int kThreads = 256, kPools = 64;

template <int PAIRS> struct CopyArgs {
    char* pool[kPools];
    int64_t page_bytes, stride;
    int32_t src[PAIRS], dst[PAIRS];
};

// Block: 256 x U words of one page (x) of one pair (y) in one pool (z).
template <typename Word, int U, int PAIRS>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyArgs<PAIRS> a) {
    char* pool = a.pool[blockIdx.z];
    const Word* s = reinterpret_cast<const Word*>(pool + a.src[blockIdx.y] * a.stride);
    Word* d = reinterpret_cast<Word*>(pool + a.dst[blockIdx.y] * a.stride);
    const int64_t n = a.page_bytes / (int64_t)sizeof(Word), i0 = (int64_t)blockIdx.x * (kThreads * U) + threadIdx.x;
    Word w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * kThreads < n) w[u] = s[i0 + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * kThreads < n) d[i0 + u * kThreads] = w[u];
}

template <typename Word, int PAIRS>
void launch(const vtx_copy_pages_params& p, int64_t pool0, int64_t pools, int64_t pair0, int64_t pairs, cudaStream_t s) {
    CopyArgs<PAIRS> a;
    for (int64_t i = 0; i < pools; ++i) a.pool[i] = static_cast<char*>(p.pool_ptrs[pool0 + i]);
    a.page_bytes = p.page_bytes; a.stride = p.page_stride_bytes;
    for (int64_t i = 0; i < pairs; ++i) { a.src[i] = (int32_t)p.src[pair0 + i]; a.dst[i] = (int32_t)p.dst[pair0 + i]; }
    const int64_t words = p.page_bytes / (int64_t)sizeof(Word);
    // four words a thread (16 KB a block) once that still gives every SM its 16 blocks; before, one
    const bool wide = ceil_div<int64_t>(words, kThreads * 4) * pairs * pools >= kNumSMs * 16;
    const dim3 grid((unsigned)ceil_div<int64_t>(words, kThreads * (wide ? 4 : 1)), (unsigned)pairs, (unsigned)pools);
    if (wide) copy_pages_kernel<Word, 4, PAIRS><<<grid, kThreads, 0, s>>>(a);
    else copy_pages_kernel<Word, 1, PAIRS><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace
}  // namespace vtx

extern "C" int vtx_copy_pages(const vtx_copy_pages_params* p, void* stream) {
    using namespace vtx;
    VTX_REQUIRE(p, VTX_ERR_BAD_ARG, "copy_pages: null pointer");
    VTX_REQUIRE(p->pools >= 0 && p->pairs >= 0 && p->num_pages >= 0 && p->page_bytes >= 0, VTX_ERR_BAD_ARG, "copy_pages: negative size");
    if (p->pools == 0 || p->pairs == 0) return VTX_OK;
    VTX_REQUIRE(p->pool_ptrs && p->src && p->dst, VTX_ERR_BAD_ARG, "copy_pages: null pointer");
    VTX_REQUIRE(p->num_pages < INT32_MAX, VTX_ERR_UNSUPPORTED, "copy_pages: more than 2^31 pages");
    VTX_REQUIRE(p->page_bytes < ((int64_t)1 << 37), VTX_ERR_UNSUPPORTED, "copy_pages: pages of more than 2^37 bytes");
    VTX_REQUIRE(p->page_stride_bytes >= p->page_bytes, VTX_ERR_BAD_ARG, "copy_pages: pages overlap");
    bool vec = p->page_bytes % 16 == 0 && p->page_stride_bytes % 16 == 0;
    for (int64_t i = 0; i < p->pools; ++i) {
        VTX_REQUIRE(p->pool_ptrs[i] || p->page_bytes == 0, VTX_ERR_BAD_ARG, "copy_pages: null pool");
        vec = vec && reinterpret_cast<uintptr_t>(p->pool_ptrs[i]) % 16 == 0;
    }
    for (int64_t i = 0; i < p->pairs; ++i)
        VTX_REQUIRE(p->src[i] >= 0 && p->src[i] < p->num_pages && p->dst[i] >= 0 && p->dst[i] < p->num_pages, VTX_ERR_BAD_ARG,
                    "copy_pages: pair %lld copies page %lld to %lld of a pool of %lld", (long long)i, (long long)p->src[i],
                    (long long)p->dst[i], (long long)p->num_pages);
    // one byte a page: 1 written, 2 read.  Pages of a call are copied at the same time, so none may be both or written twice.
    unsigned char* seen = static_cast<unsigned char*>(calloc((size_t)p->num_pages, 1));
    VTX_REQUIRE(seen, VTX_ERR_LAUNCH, "copy_pages: out of host memory");
    int64_t bad = -1;
    for (int64_t i = 0; i < p->pairs && bad < 0; ++i) {
        if (seen[p->dst[i]]) bad = p->dst[i];
        seen[p->dst[i]] = 1;
    }
    for (int64_t i = 0; i < p->pairs && bad < 0; ++i)
        if (seen[p->src[i]]) bad = p->src[i];
    free(seen);
    VTX_REQUIRE(bad < 0, VTX_ERR_BAD_ARG, "copy_pages: page %lld is written twice, or both read and written", (long long)bad);
    if (p->page_bytes == 0) return VTX_OK;
    constexpr int kFew = 32, kMany = 2048;                 // (1.3 and 17 KB of parameters)
    long long launches = 0;
    for (int64_t z = 0; z < p->pools; z += kPools) {
        const int64_t pools = p->pools - z < kPools ? p->pools - z : kPools;
        for (int64_t y = 0; y < p->pairs;) {
            const int64_t left = p->pairs - y, n = left < kMany ? left : kMany;
            if (n <= kFew) {
                if (vec) launch<uint4, kFew>(*p, z, pools, y, n, (cudaStream_t)stream);
                else launch<unsigned char, kFew>(*p, z, pools, y, n, (cudaStream_t)stream);
            } else {
                if (vec) launch<uint4, kMany>(*p, z, pools, y, n, (cudaStream_t)stream);
                else launch<unsigned char, kMany>(*p, z, pools, y, n, (cudaStream_t)stream);
            }
            y += n;
            ++launches;
        }
    }
    return check_launch("copy_pages", launches);
}
