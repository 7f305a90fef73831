// Which pages of its request a decoding row reads, for each kv head: the `first` first and the `recent` last ones, and of those between them the ones whose keys
// can score highest.  A page's score is the most that q . k can be for any key inside the page's bounds (packed.cu), for the best of the query heads that share
// the kv head:
//     score = max over heads of  sum over features of  max(q lo, q hi)  =  sum of  max(q, 0) hi + min(q, 0) lo.
//
// The sums run in 64 bits and are rounded to 32 once: of products of bfloat16 they are exact but for the last few bits of 64, so the scores, and with them the
// order, do not hang on the order of the sum; equal scores go to the lower page.  A score that is no number counts as the largest one.
//
// A cluster of CTAs takes one (row, kv head), a CTA a part of the pages, four lanes a page (a quarter of the features each) and as many
// pages at once as lanes allow, because the 64-bit chain of a page is long (2,000 pages in CTAs of 256 threads, two pages a lane: 41 us); the scores go to the first CTA's shared memory, which finds the border by halving: how many scores
// reach a threshold, bit by bit from the first that differs, until exactly as many do as are wanted or no bit is left.  (Counting 8 bits at a time with
// shared-memory atomics put nearly every score of a row into one counter, one after the other: 49 us for 16 rows and heads of 2,000 pages, of which the
// scores took some 15.)  Bound by latency where there are few rows, else by the 64-bit units (two multiply-adds a feature and head).
#include <type_traits>

#include "packed.cuh"

namespace bg {

constexpr int PS_THREADS = 512, PS_CLUSTER = 8, PS_HEADS = 8;      // (the most CTAs of a cluster; query heads at a time)
constexpr int PS_FLOATS = 50000;           // the most pages: their scores are in shared memory

// What a call brings; the host side packs the fields in their order.
struct PsParams {
    const void* q; long long q_stride;
    const unsigned char* pool; long long block_bytes;
    const int* table; const int* positions;
    int* out; unsigned* status;
    int dtype, num_pages, page_size, max_pages, T, nh, nkv, hd, top, first, recent;
    int pages_most;                    // bounds the pages of every row
};

// Ordered as the scores are, as a whole number; both noughts are one.
__device__ __forceinline__ unsigned ps_key(float s) {
    const unsigned b = __float_as_uint(s + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename TQ, int HD>
__global__ void __launch_bounds__(PS_THREADS) packed_select_kernel(const PsParams p) {
    constexpr int CHUNKS = HD / 8, MINE = CHUNKS / 4;  // pieces of 8 features of a page's bounds, and those of a lane
    extern __shared__ __align__(16) float scores[];
    __shared__ double2 q_s[CHUNKS][PS_HEADS * 8 + 1];  // (max(q, 0), min(q, 0)); the odd piece keeps four lanes' reads apart
    __shared__ unsigned ends_s[2][PS_THREADS / 32];
    __shared__ int counts[32];                         // of every bit
    pdl_launch();
    const int row = blockIdx.x, kvh = blockIdx.y, rank = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    const int pos = p.positions[row], pages = pos < 0 ? 0 : min(pos / p.page_size + 1, p.pages_most);
    const int group = p.nh / p.nkv;
    const long long bounds_at = (long long)(p.page_size / PK_TILE) * Packed<HD>::TILE;
    int* out = p.out + ((size_t)row * p.nkv + kvh) * p.top;
    if (pages <= p.top) {                              // (every CTA of the cluster: nobody waits for another)
        if (rank == 0)
            for (int i = tid; i < p.top; i += PS_THREADS) out[i] = i < pages ? i : -1;
        return;
    }
    cluster_arrive_relaxed();                          // (the first CTA has begun before its memory is written)
    cluster_wait();
    const int each = (pages + (int)gridDim.z - 1) / (int)gridDim.z, from = rank * each, to = min(pages, from + each);
    const unsigned there = peer_addr(smem_u32(scores), 0);
    for (int h0 = 0; h0 < group; h0 += PS_HEADS) {
        __syncthreads();
        for (int i = tid; i < PS_HEADS * HD; i += PS_THREADS) {
            const int h = i / HD, f = i % HD;
            const double v = h0 + h < group
                ? (double)to_float(reinterpret_cast<const TQ*>(p.q)[(size_t)row * p.q_stride + (size_t)(kvh * group + h0 + h) * HD + f]) : 0.0;
            q_s[f / 8][f % 8 * PS_HEADS + h] = make_double2(v > 0.0 ? v : 0.0, v > 0.0 ? 0.0 : v);
        }
        __syncthreads();
        const int heads = min(PS_HEADS, group - h0), quarter = tid & 3;
        auto score = [&](auto heads_) {                // (the 64-bit units are what this waits for: heads that are not there cost nothing)
        constexpr int HEADS = decltype(heads_)::value;
        for (int i0 = from; i0 + tid / 32 * 8 < to; i0 += PS_THREADS / 4) {        // (a warp without a page is done)
            const int index = i0 + tid / 4;
            const int page = index < to && index < p.max_pages ? p.table[(size_t)row * p.max_pages + index] : -1;
            const bool bad = page < 0 || page >= p.num_pages;
            const uint4* ends = reinterpret_cast<const uint4*>(p.pool + ((size_t)(bad ? 0 : page) * p.nkv + kvh) * p.block_bytes + bounds_at);
            double acc[HEADS] = {};
#pragma unroll
            for (int c = 0; c < MINE; ++c) {
                const uint4 lo4 = ends[quarter + 4 * c], hi4 = ends[CHUNKS + quarter + 4 * c];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned a = e < 2 ? lo4.x : e < 4 ? lo4.y : e < 6 ? lo4.z : lo4.w;
                    const unsigned b = e < 2 ? hi4.x : e < 4 ? hi4.y : e < 6 ? hi4.z : hi4.w;
                    const double lo = (double)__uint_as_float(e & 1 ? a & 0xffff0000u : a << 16);
                    const double hi = (double)__uint_as_float(e & 1 ? b & 0xffff0000u : b << 16);
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        const double2 w = q_s[quarter + 4 * c][e * PS_HEADS + h];
                        acc[h] = fma(w.x, hi, fma(w.y, lo, acc[h]));
                    }
                }
            }
            float best = -INFINITY;
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 1);
                acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 2);
                float s = (float)acc[h];
                if (!(s <= 3.4028234e38f)) s = 3.4028234e38f;
                if (h < heads) best = fmaxf(best, s);
            }
            if (index >= to || quarter) continue;
            if (bad) {
                best = -INFINITY;
                if (p.status) atomicOr(p.status, BG_STATUS_BAD_PAGE);
            }
            if (index < p.first || index >= pages - p.recent) best = INFINITY;
            const unsigned at = there + (unsigned)index * 4u;
            if (h0) {                                  // the best of the heads before: this thread's own store
                float old;
                asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(old) : "r"(at) : "memory");
                best = fmaxf(best, old);
            }
            st_cluster(at, best);
        }
        };
        if (heads <= 2) score(std::integral_constant<int, 2>{});
        else if (heads <= 4) score(std::integral_constant<int, 4>{});
        else if (heads <= 6) score(std::integral_constant<int, 6>{});
        else score(std::integral_constant<int, 8>{});
    }
    cluster_sync_all();
    if (rank) return;

    // ---- the border: the largest threshold that at least `top` of the ordered scores reach
    unsigned* keys = reinterpret_cast<unsigned*>(scores);
    unsigned all = 0xffffffffu, any = 0;
    for (int i = tid; i < pages; i += PS_THREADS) {
        const unsigned k = ps_key(scores[i]);
        keys[i] = k;
        all &= k; any |= k;
    }
    all = __reduce_and_sync(0xffffffffu, all);
    any = __reduce_or_sync(0xffffffffu, any);
    if (lane == 0) { ends_s[0][warp] = all; ends_s[1][warp] = any; }
    if (tid < 32) counts[tid] = 0;
    __syncthreads();
    for (int w = 0; w < PS_THREADS / 32; ++w) { all &= ends_s[0][w]; any |= ends_s[1][w]; }
    const int bits = 32 - __clz(all ^ any);            // the bits that are not the same in all of them
    unsigned border = bits >= 32 ? 0u : all >> bits << bits;
    int reached = pages;                               // how many scores reach the border
    for (int bit = bits - 1; bit >= 0 && reached != p.top; --bit) {
        const unsigned next = border | 1u << bit;
        int n = 0;
        for (int i = tid; i < pages; i += PS_THREADS) n += keys[i] >= next;
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0 && n) atomicAdd(&counts[bit], n);
        __syncthreads();
        n = counts[bit];
        if (n >= p.top) { border = next; reached = n; }
    }
    // Where exactly `top` scores reach it, all of them are taken.  Else every bit is settled and the border is a score itself: of its equals the first ones.
    // ---- the list: every page above the border and the first `want` at it, in order; a thread takes a run of pages
    const bool whole = reached == p.top;
    const int run = (pages + PS_THREADS - 1) / PS_THREADS, i0 = min(pages, tid * run), i1 = min(pages, i0 + run);
    unsigned above = 0, at = 0;
    for (int i = i0; i < i1; ++i) {
        above += whole ? keys[i] >= border : keys[i] > border;
        at += !whole && keys[i] == border;
    }
    const unsigned both = above << 16 | at;            // (fewer than 65,536 pages)
    unsigned upto = both;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) ends_s[0][warp] = upto;
    __syncthreads();
    unsigned total = 0;
#pragma unroll
    for (int w = 0; w < PS_THREADS / 32; ++w) {
        if (w < warp) upto += ends_s[0][w];
        total += ends_s[0][w];
    }
    upto -= both;
    const unsigned want = p.top - (total >> 16);       // of those at the border
    unsigned n_above = upto >> 16, n_at = upto & 0xffffu;
    for (int i = i0; i < i1; ++i) {
        const bool over = whole ? keys[i] >= border : keys[i] > border, equal = !whole && keys[i] == border;
        if (over || (equal && n_at < want)) out[n_above + min(n_at, want)] = i;
        n_above += over; n_at += equal;
    }
}

template <typename TQ, int HD>
static int ps_launch(const PsParams& p, cudaStream_t stream) {
    const size_t smem = (size_t)p.pages_most * 4;
    cudaError_t e = smem_limit(packed_select_kernel<TQ, HD>, smem);
    if (e != cudaSuccess) return (int)e;
    // as many CTAs a (row, kv head) as one an SM gives all of them at once
    int ctas = PS_CLUSTER;
    while (ctas > 1 && (long long)p.T * p.nkv * ctas > sm_count()) ctas /= 2;
    e = launch_cluster(packed_select_kernel<TQ, HD>, dim3(p.T, p.nkv, ctas), dim3(PS_THREADS), smem, stream, ctas, p);
    return e == cudaSuccess ? BG_OK : (int)e;
}

}  // namespace bg

using namespace bg;

extern "C" int bg_packed_select_most() { return PS_FLOATS; }

extern "C" int bg_packed_select_bytes() { return (int)sizeof(PsParams); }

// out[row][kv head][top]: the pages that row `row` (of request `row`) reads, ascending, -1 behind them.
extern "C" int bg_packed_select(const void* call, cudaStream_t stream) {
    const PsParams& p = *(const PsParams*)call;
    if (p.hd != 64 && p.hd != 128) return BG_ERR_UNSUPPORTED;
    if (p.T <= 0) return BG_OK;
    if (p.page_size <= 0 || p.page_size % PK_TILE || p.nkv <= 0 || p.nkv > 65535 || p.nh <= 0 || p.nh % p.nkv || p.num_pages <= 0 || p.max_pages <= 0) return BG_ERR_SHAPE;
    if (p.block_bytes % 16 || p.block_bytes < p.page_size / PK_TILE * packed_tile_bytes(p.hd) + 4 * p.hd || (uintptr_t)p.pool % 16) return BG_ERR_ALIGN;
    if (p.top <= 0 || p.first < 0 || p.recent < 1 || p.first + p.recent > p.top || p.pages_most <= 0) return BG_ERR_SHAPE;
    if (p.pages_most > PS_FLOATS) return BG_ERR_UNSUPPORTED;
    BG_DISPATCH_DTYPE(p.dtype, TQ, return p.hd == 64 ? (ps_launch<TQ, 64>(p, stream)) : (ps_launch<TQ, 128>(p, stream)));
}
