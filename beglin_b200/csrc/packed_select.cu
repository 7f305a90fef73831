// Which pages of its request a decoding row reads, for each kv head: the `first` first and the `recent` last ones, and of those between them the ones whose keys
// can score highest.  A page's score is the most that q . k can be for any key inside the page's bounds (packed.cu), for the best of the query heads that share
// the kv head (the bounds are rounded to the nearest, so that a key may lie outside by up to 2^-8 of a feature: the score orders pages, it proves nothing):
//     score = max over heads of  sum over features of  max(q lo, q hi)  =  sum of  max(q, 0) hi + min(q, 0) lo.
//
// The choice is that of sums in 64 bits, rounded to 32 once: of products of bfloat16 they are exact but for the last few bits of 64, so the order does not hang
// on the order of the sum; equal scores go to the lower page.  A score that is no number counts as the largest one.  But 64 bits are only needed next to the
// border: every page gets its score in 32 bits with a bound E on how far off that may be, and
// with A the `top`-th largest of these scores and M the largest bound, a page over A + M + E is in, one under A - M - E is out, and those between, a handful, get
// their sums in 64 bits.  (All of them in 64 bits: 50 us for 16 rows and heads of 2,000 pages, whose 64-bit multiply-adds alone take 7 and whose reads of
// the queries from shared memory as much again.)  The sums in 32 bits are products of the tensor cores, mma.sync m16n8k16 with 16 pages' bounds as they lie as the
// left operand and 8 heads' max(q, 0) and min(q, 0) as the right one; the same with the larger magnitude of both bounds and |q| gives the sum of magnitudes.
// 16 additions to an accumulator that is cut off make 2^-18 of that, E is 2^-16; queries in float are rounded to bfloat16 for this, E is then 2^-8.  (By float
// units, four lanes a page: 10 us for 256 pages of a CTA, of instructions.)
//
// A cluster of CTAs takes one (row, kv head), a CTA a part of the pages, a warp 16 of them at a time; the scores go to the first CTA's shared
// memory, which finds a border by quartering: how many scores reach a threshold, two bits a round from the first that differs, until exactly as many do as are
// wanted or no bit is left.  (Counting 8 bits at a time with shared-memory atomics put nearly every score into one counter, one after the other.)
// Bound by latency: three meetings of the cluster and two searches for a border.  4 rows of 131,072 positions, 4 kv heads, pages of 64: 20 us, an eighth of them its reads.
#include "packed.cuh"

namespace bg {

constexpr int PS_THREADS = 256, PS_WARPS = PS_THREADS / 32, PS_CLUSTER = 8, PS_HEADS = 8, PS_PAGES = 16;       // (the most CTAs of a cluster; heads and pages of a product)
constexpr int PS_MOST = 36000;             // the most pages: their scores are in shared memory
constexpr float PS_LARGEST = 3.4028234e38f;

// What a call brings; the host side packs the fields in their order.
struct PsParams {
    const void* q; long long q_stride;
    const unsigned char* pool; long long block_bytes;
    const int* table; const int* positions;
    const int* blocks;                 // [T][3]: request, row (, 1); null: i and i
    int* out; unsigned* status;
    int dtype, num_pages, page_size, max_pages, n_req, T, nh, nkv, hd, top, first, recent;
    int pages_most;                    // bounds the pages of every row
    int pad;
};

// Ordered as the scores are, as a whole number; both noughts are one.
__device__ __forceinline__ unsigned ps_key(float s) {
    const unsigned b = __float_as_uint(s + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float ps_score(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ void ps_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ps_store(unsigned addr, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(addr), "r"(v) : "memory"); }

// The largest threshold that at least `top` of the keys reach, or one that exactly `top` of them reach (then `exactly`), two bits a round.  All threads; a
// thread has up to PS_KEYS keys in registers (more are read again from shared memory: one read behind the other was most of a round).  `room` holds
// 2 * PS_WARPS + 32 numbers.
constexpr int PS_KEYS = 8;
struct PsBorder { unsigned at; bool exactly; };
__device__ __forceinline__ PsBorder ps_border(const unsigned* keys, int n, int top, unsigned* room) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool few = n <= PS_KEYS * PS_THREADS;
    unsigned k[PS_KEYS], all = 0xffffffffu, any = 0;
#pragma unroll
    for (int j = 0; j < PS_KEYS; ++j) {
        const int i = tid + j * PS_THREADS;
        k[j] = i < n ? keys[i] : 0u;                   // (no threshold is nought)
        if (i < n) { all &= k[j]; any |= k[j]; }
    }
    for (int i = tid + PS_KEYS * PS_THREADS; i < n; i += PS_THREADS) { all &= keys[i]; any |= keys[i]; }
    all = __reduce_and_sync(0xffffffffu, all);
    any = __reduce_or_sync(0xffffffffu, any);
    __syncthreads();                                   // (the room's last use)
    if (lane == 0) { room[warp] = all; room[PS_WARPS + warp] = any; }
    if (tid < 32) room[2 * PS_WARPS + tid] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PS_WARPS; ++w) { all &= room[w]; any |= room[PS_WARPS + w]; }
    const int bits = (32 - __clz(all ^ any) + 1) / 2 * 2;              // the bits that are not the same in all of them, in pairs
    unsigned border = bits >= 32 ? 0u : all >> bits << bits;
    int reached = n;
    for (int bit = bits - 2; bit >= 0 && reached != top; bit -= 2) {
        unsigned low = 0, high = 0;                    // how many reach the border with 1 (low half) and 2, and with 3, in these two bits
        const unsigned t1 = border | 1u << bit, t2 = border | 2u << bit, t3 = border | 3u << bit;
#pragma unroll
        for (int j = 0; j < PS_KEYS; ++j) {
            low += (k[j] >= t1 ? 1u : 0u) + (k[j] >= t2 ? 0x10000u : 0u);
            high += k[j] >= t3 ? 1u : 0u;
        }
        if (!few)
            for (int i = tid + PS_KEYS * PS_THREADS; i < n; i += PS_THREADS) {
                const unsigned v = keys[i];
                low += (v >= t1 ? 1u : 0u) + (v >= t2 ? 0x10000u : 0u);
                high += v >= t3 ? 1u : 0u;
            }
        low = __reduce_add_sync(0xffffffffu, low);     // (fewer than 65,536 keys)
        high = __reduce_add_sync(0xffffffffu, high);
        if (lane < 2) atomicAdd(&room[2 * PS_WARPS + bit + lane], lane ? high : low);
        __syncthreads();
        low = room[2 * PS_WARPS + bit]; high = room[2 * PS_WARPS + bit + 1];
        const int c1 = (int)(low & 0xffffu), c2 = (int)(low >> 16), c3 = (int)high;
        if (c3 >= top) { border = t3; reached = c3; }
        else if (c2 >= top) { border = t2; reached = c2; }
        else if (c1 >= top) { border = t1; reached = c1; }
    }
    return {border, reached == top};
}

template <typename TQ, int HD>
__global__ void __launch_bounds__(PS_THREADS, 2) packed_select_kernel(const PsParams p) {
    constexpr int CHUNKS = HD / 32;                    // runs of 32 features, a lane 8 of each: two steps of a product
    constexpr bool F32 = sizeof(TQ) == 4;
    extern __shared__ __align__(16) unsigned keys[];   // the first CTA's: of every page; then this CTA's own (score, bound)
    __shared__ unsigned room[2 * PS_WARPS + 32];
    __shared__ float far_of[PS_CLUSTER], cut[2], scratch[32];
    __shared__ int unsure[PS_THREADS], n_unsure;
    pdl_launch();
    const int item = blockIdx.x, kvh = blockIdx.y, rank = blockIdx.z, ranks = gridDim.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    const int req = p.blocks ? p.blocks[3 * item] : item, row = p.blocks ? p.blocks[3 * item + 1] : item;
    const int pos = p.positions[row], pages = pos < 0 ? 0 : min(pos / p.page_size + 1, p.pages_most);
    const int group = p.nh / p.nkv;
    const long long bounds_at = (long long)(p.page_size / PK_TILE) * Packed<HD>::TILE;
    int* out = p.out + ((size_t)item * p.nkv + kvh) * p.top;
    if (pages <= p.top) {                              // (every CTA of the cluster: nobody waits for another)
        if (rank == 0)
            for (int i = tid; i < p.top; i += PS_THREADS) out[i] = i < pages ? i : -1;
        return;
    }
    cluster_arrive_relaxed();                          // (the others have begun before their memory is written)
    cluster_wait();
    const int each = (pages + ranks - 1) / ranks, from = rank * each, to = min(pages, from + each);
    float2* mine = reinterpret_cast<float2*>(keys + (p.pages_most + 1) / 2 * 2);       // [each]: a page's score in 32 bits, and how far off it may be
    const unsigned there = peer_addr(smem_u32(keys), 0);
    const TQ* q = reinterpret_cast<const TQ*>(p.q) + (size_t)row * p.q_stride + (size_t)kvh * group * HD;
    // the bounds of a page, or null where the table names none
    auto bounds_of = [&](int index) -> const unsigned char* {
        const int page = index < p.max_pages && req >= 0 && req < p.n_req ? p.table[(size_t)req * p.max_pages + index] : -1;
        return page >= 0 && page < p.num_pages ? p.pool + ((size_t)page * p.nkv + kvh) * p.block_bytes + bounds_at : nullptr;
    };

    // ---- every page's score in 32 bits
    float far = 0.0f;                                  // the largest bound
    const int g = lane >> 2, t = lane & 3;
    for (int h0 = 0; h0 < group; h0 += PS_HEADS) {
        const int heads = min(PS_HEADS, group - h0);
        unsigned above[CHUNKS][4], below[CHUNKS][4], size[CHUNKS][4];           // max(q, 0), min(q, 0), |q| of head g
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            float v[8] = {};
            if (g < heads) load8(q + (size_t)(h0 + g) * HD + 32 * c + 8 * t, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                const unsigned bits = *reinterpret_cast<const unsigned*>(&x);
                const unsigned negative = ((bits >> 15) & 0x00010001u) * 0xffffu;
                above[c][i] = bits & ~negative; below[c][i] = bits & negative; size[c][i] = bits & 0x7fff7fffu;
            }
        }
        for (int i0 = from + warp * PS_PAGES; i0 < to; i0 += PS_WARPS * PS_PAGES) {
            int index[2];
            const unsigned char* ends[2];              // pages g and g + 8
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                index[n] = i0 + 8 * n + g;
                ends[n] = index[n] < to ? bounds_of(index[n]) : nullptr;
            }
            uint4 lo[CHUNKS][2], hi[CHUNKS][2];
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const uint4* at = reinterpret_cast<const uint4*>(ends[n] ? ends[n] : p.pool + bounds_at) + 4 * c + t;
                    lo[c][n] = at[0]; hi[c][n] = at[HD / 8];
                }
            float s[4] = {}, sum[4] = {};              // (page g, heads 2t and 2t + 1; page g + 8)
            auto most = [](unsigned a, unsigned b) {   // the larger magnitude of two pairs
                const unsigned x = a & 0x7fff7fffu, y = b & 0x7fff7fffu;
                return __vmaxu2(x, y);                 // (magnitudes are ordered as whole numbers)
            };
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const unsigned l[2][4] = {{lo[c][0].x, lo[c][0].y, lo[c][0].z, lo[c][0].w}, {lo[c][1].x, lo[c][1].y, lo[c][1].z, lo[c][1].w}};
                const unsigned u[2][4] = {{hi[c][0].x, hi[c][0].y, hi[c][0].z, hi[c][0].w}, {hi[c][1].x, hi[c][1].y, hi[c][1].z, hi[c][1].w}};
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    ps_mma(s, u[0][k], u[1][k], u[0][k + 1], u[1][k + 1], above[c][k], above[c][k + 1]);
                    ps_mma(s, l[0][k], l[1][k], l[0][k + 1], l[1][k + 1], below[c][k], below[c][k + 1]);
                    ps_mma(sum, most(l[0][k], u[0][k]), most(l[1][k], u[1][k]), most(l[0][k + 1], u[0][k + 1]), most(l[1][k + 1], u[1][k + 1]),
                           size[c][k], size[c][k + 1]);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float best = -INFINITY, bound = 0.0f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float a = s[2 * n + j], b = sum[2 * n + j];
                    if (2 * t + j >= heads) continue;
                    if (!(b < 1e37f) || a != a) { a = 0.0f; b = INFINITY; }      // (beyond what 32 bits hold, or no number)
                    best = fmaxf(best, a); bound = fmaxf(bound, (F32 ? 0x1p-8f : 0x1p-16f) * b);
                }
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
                    bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, d));
                }
                if (index[n] >= to || t) continue;
                if (!ends[n]) {
                    best = -INFINITY; bound = 0.0f;
                    if (p.status) atomicOr(p.status, BG_STATUS_BAD_PAGE);
                }
                float2& have = mine[index[n] - from];
                if (h0) { best = fmaxf(best, have.x); bound = fmaxf(bound, have.y); }
                have = make_float2(best, bound);
                const bool always = index[n] < p.first || index[n] >= pages - p.recent;
                if (!always) far = fmaxf(far, bound);
                if (h0 + PS_HEADS >= group) ps_store(there + 4u * (unsigned)index[n], ps_key(always ? INFINITY : best));
            }
        }
    }
    far = block_max(far, scratch);
    if (tid == 0) {
        n_unsure = 0;
        st_cluster(peer_addr(smem_u32(&far_of[rank]), 0), far);
    }
    cluster_sync_all();

    // ---- the `top`-th largest of them, and the largest bound, for all CTAs
    if (rank == 0) {
        const PsBorder b = ps_border(keys, pages, p.top, room);
        unsigned least = 0xffffffffu;                  // (where exactly `top` scores reach the border, it is the least of those)
        for (int i = tid; i < pages; i += PS_THREADS)
            if (keys[i] >= b.at) least = min(least, keys[i]);
        least = __reduce_min_sync(0xffffffffu, least);
        __syncthreads();
        if (lane == 0) room[warp] = least;
        __syncthreads();
        if (tid < ranks) {
            for (int w = 0; w < PS_WARPS; ++w) least = min(least, room[w]);
            float most = 0.0f;
            for (int r = 0; r < ranks; ++r) most = fmaxf(most, far_of[r]);
            st_cluster(peer_addr(smem_u32(&cut[0]), (unsigned)tid), ps_score(least));
            st_cluster(peer_addr(smem_u32(&cut[1]), (unsigned)tid), most);
        }
    }
    cluster_sync_all();

    // ---- what is in, what is out, and the sums in 64 bits of what is between
    const float middle = cut[0], most = cut[1];
    for (int i0 = from; i0 < to; i0 += PS_THREADS) {
        const int index = i0 + tid;
        if (index < to) {
            const float2 have = mine[index - from];
            const bool always = index < p.first || index >= pages - p.recent;
            if (always || have.x - have.y > middle + most) ps_store(there + 4u * (unsigned)index, 0xffffffffu);
            else if (have.x + have.y < middle - most) ps_store(there + 4u * (unsigned)index, 0u);
            else unsure[atomicAdd(&n_unsure, 1)] = index;            // (their order is nobody's business)
        }
        __syncthreads();
        const int n = n_unsure;
        for (int i = warp; i < n; i += PS_WARPS) {
            constexpr int PER = HD / 32;               // features of a lane
            const unsigned char* ends = bounds_of(unsure[i]);
            float best = -INFINITY;
            if (ends) {
                double lo[PER], hi[PER];
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    lo[e] = (double)__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(ends)[lane * PER + e]);
                    hi[e] = (double)__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(ends)[HD + lane * PER + e]);
                }
                for (int h = 0; h < group; ++h) {
                    double a = 0.0;
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        const double v = (double)to_float(q[(size_t)h * HD + lane * PER + e]);
                        a = fma(v > 0.0 ? v : 0.0, hi[e], fma(v > 0.0 ? 0.0 : v, lo[e], a));
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
                    float s = (float)a;
                    if (!(s <= PS_LARGEST)) s = PS_LARGEST;
                    best = fmaxf(best, s);
                }
            }
            if (lane == 0) ps_store(there + 4u * (unsigned)unsure[i], ps_key(best));     // (between nought and the largest number)
        }
        __syncthreads();
        if (tid == 0) n_unsure = 0;
        __syncthreads();
    }
    cluster_sync_all();
    if (rank) return;

    // ---- the list: every page above the border and the first ones at it, in order; a thread takes a run of pages
    const PsBorder b = ps_border(keys, pages, p.top, room);
    const int run = (pages + PS_THREADS - 1) / PS_THREADS, i0 = min(pages, tid * run), i1 = min(pages, i0 + run);
    unsigned above = 0, at = 0;
    for (int i = i0; i < i1; ++i) {
        above += b.exactly ? keys[i] >= b.at : keys[i] > b.at;
        at += !b.exactly && keys[i] == b.at;
    }
    const unsigned both = above << 16 | at;            // (fewer than 65,536 pages)
    unsigned upto = both;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    __syncthreads();
    if (lane == 31) room[warp] = upto;
    __syncthreads();
    unsigned total = 0;
#pragma unroll
    for (int w = 0; w < PS_WARPS; ++w) {
        if (w < warp) upto += room[w];
        total += room[w];
    }
    upto -= both;
    const unsigned want = p.top - (total >> 16);       // of those at the border
    unsigned n_above = upto >> 16, n_at = upto & 0xffffu;
    for (int i = i0; i < i1; ++i) {
        const bool over = b.exactly ? keys[i] >= b.at : keys[i] > b.at, equal = !b.exactly && keys[i] == b.at;
        if (over || (equal && n_at < want)) out[n_above + min(n_at, want)] = i;
        n_above += over; n_at += equal;
    }
}

template <typename TQ, int HD>
static int ps_launch(const PsParams& p, cudaStream_t stream) {
    // as many CTAs a (row, kv head) as two an SM give all of them at once, and at least as many as hold the scores of the pages (4 kv heads, us by this rule, always 8, and as
    // few as hold them: 4 rows of 131,072 positions 20.9, 21.2, 42.4; 16 rows of 32,000 19.1, 35.5, 24.7; 64 rows of 8,000 16.5, 93.6, 16.5)
    auto bytes = [&](int ctas) { return (size_t)(p.pages_most + 1) / 2 * 8 + (size_t)((p.pages_most + ctas - 1) / ctas) * 8; };
    int ctas = PS_CLUSTER;
    while (ctas > 1 && (long long)p.T * p.nkv * ctas > 2LL * sm_count() && bytes(ctas / 2) <= 100 * 1024) ctas /= 2;
    const size_t smem = bytes(ctas);
    cudaError_t e = smem_limit(packed_select_kernel<TQ, HD>, smem);
    if (e != cudaSuccess) return (int)e;
    e = launch_cluster(packed_select_kernel<TQ, HD>, dim3(p.T, p.nkv, ctas), dim3(PS_THREADS), smem, stream, ctas, p);
    return e == cudaSuccess ? BG_OK : (int)e;
}

}  // namespace bg

using namespace bg;

extern "C" int bg_packed_select_most() { return PS_MOST; }

extern "C" int bg_packed_select_bytes() { return (int)sizeof(PsParams); }

// out[i][kv head][top]: the pages that the i-th row of `blocks` (or row i, of request i) reads, ascending, -1 behind them.
extern "C" int bg_packed_select(const void* call, cudaStream_t stream) {
    const PsParams& p = *(const PsParams*)call;
    if (p.hd != 64 && p.hd != 128) return BG_ERR_UNSUPPORTED;
    if (p.T <= 0) return BG_OK;
    if (p.page_size <= 0 || p.page_size % PK_TILE || p.nkv <= 0 || p.nkv > 65535 || p.nh <= 0 || p.nh % p.nkv || p.num_pages <= 0 || p.max_pages <= 0) return BG_ERR_SHAPE;
    if (p.block_bytes % 16 || p.block_bytes < p.page_size / PK_TILE * packed_tile_bytes(p.hd) + 4 * p.hd || (uintptr_t)p.pool % 16
        || ((long long)(uintptr_t)p.q | p.q_stride * (p.dtype == BG_DTYPE_F32 ? 4 : 2)) % 16) return BG_ERR_ALIGN;
    if (p.top <= 0 || p.first < 0 || p.recent < 1 || p.first + p.recent > p.top || p.pages_most <= 0) return BG_ERR_SHAPE;
    if (p.pages_most > PS_MOST) return BG_ERR_UNSUPPORTED;
    BG_DISPATCH_DTYPE(p.dtype, TQ, return p.hd == 64 ? (ps_launch<TQ, 64>(p, stream)) : (ps_launch<TQ, 128>(p, stream)));
}
