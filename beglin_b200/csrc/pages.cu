// Copies of the first positions of pages, for all stages of a pool at once: what a request needs of another's last page when it goes on
// from the same text by itself.
//
// A page is `outer` blocks of `rows` positions of `bytes` bytes (keys and values of every kv head; one block for a latent); the first `n`
// positions of every block are copied.  A thread takes one piece of 16 bytes (less where sizes or addresses ask for it) of a source page and
// writes it to up to PAGES_EACH of the pages that get it (a source comes from the L2 again for the next ones).  Bound by the bytes written: 45 positions of
// 28 stages of 64 KB pages to 63 pages, 81 MB, 14.2 us with four targets a thread (floor 12.6), 15.4 with two, 14.5 with eight, 23.3 with all of them.
#include "common.cuh"

namespace bg {

constexpr int PAGES_MOST = 224;            // pairs of a launch: they travel as the kernel's argument
constexpr int PAGES_THREADS = 256, PAGES_EACH = 4;
struct PageCopies {
    int count, groups;
    int first[PAGES_MOST + 1];             // where a group's targets begin
    int src[PAGES_MOST], dst[PAGES_MOST];  // a group's source; targets
};

template <typename T>
__global__ void __launch_bounds__(PAGES_THREADS) copy_pages_kernel(unsigned char* pool, long long stage_bytes, long long page_bytes, long long block_bytes,
                                                                   int per_block, long long pieces, const __grid_constant__ PageCopies c) {
    // (no early start for what comes behind: the attention kernels ask for older positions before they wait for the kernel ahead of them, and these are older)
    pdl_wait();
    const long long at = (long long)blockIdx.x * PAGES_THREADS + threadIdx.x;
    if (at >= pieces) return;
    const long long o = at / per_block;
    unsigned char* stage = pool + (size_t)blockIdx.z * stage_bytes + o * block_bytes + (at - o * per_block) * (long long)sizeof(T);
    const int g = blockIdx.y;
    const T v = *reinterpret_cast<const T*>(stage + (size_t)c.src[g] * page_bytes);
    for (int i = c.first[g]; i < c.first[g + 1]; ++i) *reinterpret_cast<T*>(stage + (size_t)c.dst[i] * page_bytes) = v;
}

template <typename T>
static int pages_launch(void* pool, int stages, long long stage_bytes, long long page_bytes, int outer, long long block_bytes, long long copy_bytes,
                        const PageCopies& c, cudaStream_t stream) {
    const long long per_block = copy_bytes / (long long)sizeof(T), pieces = per_block * outer;
    const long long blocks = (pieces + PAGES_THREADS - 1) / PAGES_THREADS;
    if (blocks > 0x7fffffffLL || per_block > 0x7fffffffLL) return BG_ERR_SHAPE;
    cudaError_t e = launch(copy_pages_kernel<T>, dim3((unsigned)blocks, (unsigned)c.groups, (unsigned)stages), dim3(PAGES_THREADS), 0, stream,
                           (unsigned char*)pool, stage_bytes, page_bytes, block_bytes, (int)per_block, pieces, c);
    return e == cudaSuccess ? BG_OK : (int)e;
}

}  // namespace bg

using namespace bg;

// The most pairs that one call takes.
extern "C" int bg_copy_pages_most() { return PAGES_MOST; }

// pages[dst[i]] <- pages[src[i]] for the first `n` of `rows` positions of `bytes` bytes in each of the `outer` blocks of a page, in all stages.  src and dst
// are host arrays, equal sources side by side; the targets differ from one another and from the sources.
extern "C" int bg_copy_pages(void* pool, int stages, long long stage_bytes, int num_pages, long long page_bytes, int outer, int rows, long long bytes, int n,
                             const int* src, const int* dst, int count, cudaStream_t stream) {
    if (count <= 0 || n == 0) return BG_OK;
    if (count > PAGES_MOST || stages <= 0 || stages > 65535 || outer <= 0 || rows <= 0 || bytes <= 0 || n < 0 || n > rows) return BG_ERR_SHAPE;
    if ((long long)outer * rows * bytes > page_bytes) return BG_ERR_SHAPE;
    PageCopies c;
    c.count = count; c.groups = 0;
    for (int i = 0; i < count; ++i) {
        if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages) return BG_ERR_SHAPE;
        if (i == 0 || src[i] != src[i - 1] || i - c.first[c.groups - 1] == PAGES_EACH) { c.src[c.groups] = src[i]; c.first[c.groups++] = i; }
        c.dst[i] = dst[i];
    }
    c.first[c.groups] = count;
    const long long block = rows * bytes, copy = n * bytes;
    const long long all = (long long)(uintptr_t)pool | stage_bytes | page_bytes | block | copy;      // (its low bits are nought where all of theirs are)
    if (all % 16 == 0) return pages_launch<uint4>(pool, stages, stage_bytes, page_bytes, outer, block, copy, c, stream);
    if (all % 4 == 0) return pages_launch<unsigned>(pool, stages, stage_bytes, page_bytes, outer, block, copy, c, stream);
    if (all % 2 == 0) return pages_launch<unsigned short>(pool, stages, stage_bytes, page_bytes, outer, block, copy, c, stream);
    return BG_ERR_ALIGN;
}
