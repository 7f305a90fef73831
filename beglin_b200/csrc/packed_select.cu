// Which pages of its request a decoding row reads, for each kv head: the `first` first and the `recent` last ones, and of those between them the ones whose keys
// can score highest.  A page's score is the most that q . k can be for any key inside the page's bounds (packed.cu), for the best of the query heads that share
// the kv head:
//     score = max over heads of  sum over features of  max(q lo, q hi)  =  sum of  max(q, 0) hi + min(q, 0) lo.
//
// The sums run in 64 bits and are rounded to 32 once: of products of bfloat16 they are exact but for the last few bits of 64, so the scores, and with them the
// order, do not hang on the order of the sum; equal scores go to the lower page.  A score that is no number counts as the largest one.
//
// A cluster of CTAs takes one (row, kv head), a CTA a part of the pages, four lanes a page (a quarter of the features each); the scores go to the first CTA's shared
// memory, which finds the border by four rounds of counting 8 bits of the ordered scores and lists the pages above it in order.  Bound by latency where there are
// few rows, else by the 64-bit units (two multiply-adds a feature and head).
#include "packed.cuh"

namespace bg {

constexpr int PS_THREADS = 256, PS_CLUSTER = 8, PS_HEADS = 8, PS_FLOATS = 50000;       // PS_FLOATS: the most pages, whose scores are in shared memory

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
    __shared__ int hist[256], sums[PS_THREADS / 32], chosen[2];
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
    const int each = (pages + PS_CLUSTER - 1) / PS_CLUSTER, from = rank * each, to = min(pages, from + each);
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
        const int heads = min(PS_HEADS, group - h0);
        for (int i0 = from; i0 < to; i0 += PS_THREADS / 4) {
            const int index = i0 + tid / 4, quarter = tid & 3;
            const bool have = index < to;
            int page = have && index < p.max_pages ? p.table[(size_t)row * p.max_pages + index] : -1;
            const bool bad = have && (page < 0 || page >= p.num_pages);
            if (bad || !have) page = 0;
            const uint4* ends = reinterpret_cast<const uint4*>(p.pool + ((size_t)page * p.nkv + kvh) * p.block_bytes + bounds_at);
            uint4 lo4[MINE], hi4[MINE];
#pragma unroll
            for (int c = 0; c < MINE; ++c) { lo4[c] = ends[quarter + 4 * c]; hi4[c] = ends[CHUNKS + quarter + 4 * c]; }
            double acc[PS_HEADS] = {};
#pragma unroll
            for (int c = 0; c < MINE; ++c) {
                const unsigned l[4] = {lo4[c].x, lo4[c].y, lo4[c].z, lo4[c].w}, u[4] = {hi4[c].x, hi4[c].y, hi4[c].z, hi4[c].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const double lo = (double)__uint_as_float(e & 1 ? l[e / 2] & 0xffff0000u : l[e / 2] << 16);
                    const double hi = (double)__uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
#pragma unroll
                    for (int h = 0; h < PS_HEADS; ++h) {
                        const double2 w = q_s[quarter + 4 * c][e * PS_HEADS + h];
                        acc[h] = fma(w.x, hi, fma(w.y, lo, acc[h]));
                    }
                }
            }
            float best = -INFINITY;
#pragma unroll
            for (int h = 0; h < PS_HEADS; ++h) {
                acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 1);
                acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 2);
                float s = (float)acc[h];
                if (!(s <= 3.4028234e38f)) s = 3.4028234e38f;
                if (h < heads) best = fmaxf(best, s);
            }
            if (bad) {
                best = -INFINITY;
                if (p.status && quarter == 0) atomicOr(p.status, BG_STATUS_BAD_PAGE);
            }
            if (index < p.first || index >= pages - p.recent) best = INFINITY;
            if (have && quarter == 0) {
                const unsigned at = there + (unsigned)index * 4u;
                if (h0) {                              // the best of the heads before: this thread's own store
                    float old;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(old) : "r"(at) : "memory");
                    best = fmaxf(best, old);
                }
                st_cluster(at, best);
            }
        }
    }
    cluster_sync_all();
    if (rank) return;

    // ---- the border: the largest key of which, with those above it, there are at least `top`
    unsigned prefix = 0;
    int want = p.top;
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < pages; i += PS_THREADS) {
            const unsigned k = ps_key(scores[i]);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[255 - (k >> shift & 255u)], 1);
        }
        __syncthreads();
        const int mine = hist[tid];
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        for (int w = 0; w < warp; ++w) upto += sums[w];
        if (upto >= want && upto - mine < want) { chosen[0] = 255 - tid; chosen[1] = want - (upto - mine); }
        __syncthreads();
        prefix |= (unsigned)chosen[0] << shift;
        want = chosen[1];
        __syncthreads();
    }
    // ---- the list: every page above the border and the first `want` at it, in order; a thread takes a run of pages
    const int run = (pages + PS_THREADS - 1) / PS_THREADS, i0 = min(pages, tid * run), i1 = min(pages, i0 + run);
    unsigned above = 0, at = 0;
    for (int i = i0; i < i1; ++i) {
        const unsigned k = ps_key(scores[i]);
        above += k > prefix; at += k == prefix;
    }
    unsigned both = above << 16 | at, upto = both;     // (fewer than 65,536 pages)
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) sums[warp] = (int)upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += (unsigned)sums[w];
    upto -= both;
    unsigned n_above = upto >> 16, n_at = upto & 0xffffu;
    for (int i = i0; i < i1; ++i) {
        const unsigned k = ps_key(scores[i]);
        const bool take = k > prefix || (k == prefix && n_at < (unsigned)want);
        if (take) out[n_above + min(n_at, (unsigned)want)] = i;
        n_above += k > prefix; n_at += k == prefix;
    }
}

template <typename TQ, int HD>
static int ps_launch(const PsParams& p, cudaStream_t stream) {
    const size_t smem = (size_t)p.pages_most * 4;
    cudaError_t e = smem_limit(packed_select_kernel<TQ, HD>, smem);
    if (e != cudaSuccess) return (int)e;
    e = launch_cluster(packed_select_kernel<TQ, HD>, dim3(p.T, p.nkv, PS_CLUSTER), dim3(PS_THREADS), smem, stream, PS_CLUSTER, p);
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
