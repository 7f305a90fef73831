// Attention over pages that hold keys and values in 4 bits (packed.cuh), for single tokens and short runs of rows: softmax(q K^T scale) V with
// K = lowest + step u, never written out.
//
// Both products run as mma.sync m16n8k16 with the CODES as the left operand.  The low byte of a bfloat16 whose upper byte is nought stands for itself times
// 2^-133 (exponents 0 and 1 share a unit), so a code needs no conversion: masked out of its word at bits 0 or 4 it IS the number u 2^-133 or 16 u 2^-133, and
// the right operand is scaled up by powers of two to meet it (two masks, a shift by 8, two masks: five operations for 8 codes; as 128 + u, 0x4300 | u, which
// needs every code at bit 0, it took seven, a product more for the 128 and, over 131,072 positions, a third of the result's last digit).  (step, lowest)
// are applied in float outside the product:
//     q . k   = sum over groups of  step (sum q u) + lowest (sum q)
//     p V     = sum over positions of  (p step) u + p lowest
//             = sum over positions of  r u - 8 r + p (lowest + 8 step),  r = p step rounded to bfloat16 (but for float queries),
// so that the only rounding of the cache's side is that of r, and it counts for u - 8 alone: 4.6 in the root of the mean of squares, where u are 8.8 (results
// 0.0021 of their norm off, with u alone 0.0029; rounding them to bfloat16 is 0.0017).  The sum of r is a product with -1; 2 us of 70.  Sums over a warp's whole range
// of positions stay in the tensor cores' accumulators, 32 bits that are cut off rather than rounded (float queries take a tile's sums out: next to what r loses that
// does not show, in float it does); 2^x and tanh are the approximate instructions, good to 22 bits, and float's own for float queries.  Keys: 16 positions
// by 16 features times features by 8 columns; values: 16 features by 16 positions times positions by columns.  A column is one (row, query head): the
// queries of a kv head are the narrow side, so 8 heads waste nothing of the product and a code is unpacked once for all of them.  The weights reach the
// second product's layout through movmatrix.  Float queries and weights go in three bfloat16 parts.
//
// Ranges: a row of queries is scaled by the power of two that brings its largest to 2^100.  Weights carry 2^64, and 2^8 where the maximum has not moved, so values
// may have steps up to 2^36 (32,768 positions of such weights), and those under 2^-50 lose digits.
//
// Why this shape: at the bandwidth of HBM a position of a kv head (144 bytes for heads of 128) has to be done in some 6 cycles of an SM, 25 warp
// instructions at best.  It takes 18 for 8 columns, half of them on the units of integers and logic, which take one every two cycles; with the queries on
// the left (16 rows, half of them empty) it took the tensor cores twice the products and the softmax twice the numbers.  4 rows of 131,072 positions, 4 kv
// heads: 70 us, 63 % of the bandwidth of a copy (some 80 % but for what does not grow with the length: a start, two kernels, where results meet); 64 rows
// of 2,048 to 8,192, 2 kv heads: 35 us, 41 %.  Bound by these instructions: with all pages in the L2 it takes 95 % of the time.  A warp has a ring of its
// own (STAGES chunks of 16 or 32 positions, one bulk copy each) and its own running maximum, sum and result, so that nothing in the loop waits for another
// warp; the warps' results meet at the end, those of a long request's ranges in packed_merge_kernel.
#include <type_traits>

#include "packed.cuh"

namespace bg {

constexpr int PA_WARPS = 8, PA_THREADS = PA_WARPS * 32, PA_STAGES = 2;
constexpr int PA_BLOCKS = 1024;            // blocks of rows whose units a CTA sums up
constexpr float PA_LOG2E = 1.4426950408889634f;

// What a call brings; the host side packs the fields in their order.
struct PaCall {
    const void* q; const unsigned char* pool;
    const int* table; const int* positions;
    const int* blocks;                 // [n][3]: request, first row, rows; null: block i is row i of request i
    const int* list;                   // [blocks][nkv][top] page indexes to read (less than 0: none), or null: all
    float* part_o; float* part_ml;     // (with ctas) [CTA][2][column][HD], [..][2]: what a CTA has of a stream that it shares with others
    void* out; const float* sink_w; unsigned* status;
    long long q_stride, block_bytes, out_stride;
    int dtype, num_pages, page_size, max_pages, n_req;
    int n, rows;                       // blocks, and the most rows of one
    int top;
    int ctas;                          // CTAs that share all streams' positions evenly; 0: none is shared so
    int cluster;                       // (without ctas) CTAs of a cluster that share a stream's positions
    int nh, nkv, hd, window, sink, pad;
    float scale, softcap;
};
struct PaParams : PaCall {
    int group, head_blocks, heads_each;            // query heads of a kv head, the blocks that they are cut into, heads of a block
    int2* shared_by;                               // [block][heads_all]: the first CTA that has a part of a stream, and how many have
    int heads_all;                                 // kv heads times head blocks: a stream is one of them of one block of rows
    float scale_log2, cap_log2, scale_over_cap;
};

// The chunks of KEYS positions that a block of rows reads: the first one, and how many (of a list, from its first entry on).
struct PaChunks { int first, count; };
__device__ __forceinline__ PaChunks pa_chunks(const PaParams& p, int keys, int row0, int rows) {
    const int pos_first = p.positions[row0], pos_last = p.positions[row0 + rows - 1];
    if (pos_last < 0) return {0, 0};
    if (p.list) return {0, min(p.top, pos_last / p.page_size + 1) * (p.page_size / keys)};
    const int first = (p.window > 0 ? max(0, pos_first - p.window + 1) : 0) / keys;
    return {first, pos_last / keys + 1 - first};
}
// ... in units of a chunk for each warp, one at least (a block without positions has results too).
__device__ __forceinline__ int pa_units(const PaParams& p, int keys, int block) {
    const int row0 = p.blocks ? p.blocks[3 * block + 1] : block, rows = p.blocks ? p.blocks[3 * block + 2] : 1;
    return max(1, (pa_chunks(p, keys, row0, rows).count + PA_WARPS - 1) / PA_WARPS);
}

__device__ __forceinline__ void pa_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pa_transposed(unsigned a) {
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ unsigned pa_pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<unsigned*>(&h);
}
constexpr float PA_UP = 64.0f;                         // weights, and sums of them, are 2^(x - maximum) times 2^PA_UP
constexpr float PA_SLACK = 8.0f;
constexpr unsigned PA_ONE = 0x00010001u;               // the code 1 of two features, at bits 0
constexpr unsigned PA_MINUS = 0xbf80bf80u;             // -1 twice
// The pair of codes at bits 4 i of both halves of a word: u 2^-133 where i is even, 16 u 2^-133 where it is odd.
__device__ __forceinline__ unsigned pa_codes(unsigned w, int i) { return (i < 2 ? w : w >> 8) & (i % 2 ? 0x00f000f0u : 0x000f000fu); }
__device__ __forceinline__ void pa_bulk_load(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float pa_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// c log2(e) tanh(x / c) of x / c.
template <bool F32>
__device__ __forceinline__ float pa_squashed(float x, float cap_log2) {
    if constexpr (F32) return cap_log2 * tanhf(x);
    float r;                                           // tanh x = 1 - 2 / (1 + e^(2 x))
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(1.0f + pa_exp2(x * (2.0f * PA_LOG2E))));
    return cap_log2 * fmaf(-2.0f, r, 1.0f);
}

template <int HD, int NT, bool F32>
struct PaShape {
    static constexpr int PARTS = F32 ? 3 : 1, COLS = 8 * NT, ROW = HD + 2;      // ROW: floats of a column's result in shared memory
    static constexpr int JOIN = PA_WARPS * COLS * (ROW + 2) * 4;
};

// SHARE: the CTAs share all streams evenly; else a stream has a CTA, or a cluster of them.  (Both in one kernel cost the first 5 % by the registers of the second.)
template <int HD, int NT, bool F32, int CT, bool SHARE>
__global__ void __launch_bounds__(PA_THREADS, NT == 1 && !F32 ? 2 : 1) packed_attention_kernel(const PaParams p) {
    using S = PaShape<HD, NT, F32>;
    using L = Packed<HD>;
    using TQ = typename std::conditional<F32, float, __nv_bfloat16>::type;
    constexpr int GROUPS = L::GROUPS, PARTS = S::PARTS, COLS = S::COLS, KEYS = CT * PK_TILE, BYTES = CT * L::TILE;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long bars[PA_WARPS][PA_STAGES];
    __shared__ int where[PA_WARPS][PA_STAGES];         // a stage's first position, or -1: nothing to read
    // units of a head's blocks in front of each block; or what a cluster's CTAs have of this one's columns
    constexpr int MEET = SHARE ? PA_BLOCKS + 1 + PA_WARPS : COLS * (HD + 2);
    __shared__ __align__(16) int before[MEET];
    __shared__ int gave_up;
    pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (threadIdx.x < PA_WARPS * PA_STAGES) mbar_init(&bars[threadIdx.x / PA_STAGES][threadIdx.x % PA_STAGES], 1);
    if (threadIdx.x == 0) gave_up = 0;
    mbar_init_fence();
    const int ranks = SHARE ? 1 : gridDim.z, rank = SHARE ? 0 : blockIdx.z;
    if (ranks > 1) cluster_arrive_relaxed();           // (the others have begun before their memory is written)
    __syncthreads();
    if (ranks > 1) cluster_wait();
    pdl_wait();
    // ---- what this CTA reads.  The streams (a kv head, or a block of its query heads, of a block of rows; the blocks of one head one behind the other) are cut
    // in units of PA_WARPS chunks, and the CTAs share the units evenly, whatever the lengths: a CTA's run of units begins and ends inside streams, whose results
    // packed_merge_kernel joins, and those that lie inside the run are finished here.  (A fixed number of CTAs for every stream left 64 rows of 2,048 to 8,192
    // positions, 2 kv heads, at 40 us for the longest ones.)  Few and short streams have a cluster each instead, whose CTAs take even parts and join them in shared
    // memory: no second kernel, no scratch.
    int unit = 0, stop = 1;                            // (the host sees to it that they fit)
    if constexpr (SHARE) {
        int mine[PA_BLOCKS / PA_THREADS], sum = 0;
#pragma unroll
        for (int i = 0; i < PA_BLOCKS / PA_THREADS; ++i) {
            const int b = threadIdx.x * (PA_BLOCKS / PA_THREADS) + i;
            mine[i] = b < p.n ? pa_units(p, KEYS, b) : 0;
            sum += mine[i];
        }
        int upto = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 31) before[PA_BLOCKS + 1 + warp] = upto;
        __syncthreads();
        int per_head = 0;
        for (int w = 0; w < PA_WARPS; ++w) {
            if (w < warp) upto += before[PA_BLOCKS + 1 + w];
            per_head += before[PA_BLOCKS + 1 + w];
        }
        upto -= sum;
        if (threadIdx.x == 0) before[PA_BLOCKS] = per_head;
#pragma unroll
        for (int i = 0; i < PA_BLOCKS / PA_THREADS; ++i) {
            before[threadIdx.x * (PA_BLOCKS / PA_THREADS) + i] = upto;
            upto += mine[i];
        }
        __syncthreads();
        const long long units = (long long)per_head * p.heads_all;
        const long long share = min((long long)p.ctas, units);          // (none without a unit: the merge counts on it)
        unit = blockIdx.x < share ? (int)(blockIdx.x * units / share) : 0;
        stop = blockIdx.x < share ? (int)((blockIdx.x + 1) * units / share) : 0;
    }
    // What is left of the stream that holds `unit`, as far as this CTA's run goes: where its copies come from, and which of them this warp waits for.
    int block, hy, u0, turns, begin, end, chunk0, req, pos_last;
    bool finished;
    const int* list;
    const int per_page = p.page_size / KEYS;
    auto next_stream = [&]() {
    block = blockIdx.x; hy = blockIdx.y;
    int u1, u_all;
    if constexpr (SHARE) {
        const int per_head = before[PA_BLOCKS];
        hy = unit / per_head;
        const int r = unit - hy * per_head;
        int low = 0, high = p.n - 1;                   // the last block that begins at or before r
        while (low < high) {
            const int mid = (low + high + 1) / 2;
            if (before[mid] <= r) low = mid;
            else high = mid - 1;
        }
        block = low;
        u_all = (block + 1 < p.n ? before[block + 1] : per_head) - before[block];
        u0 = r - before[block];
        u1 = min(u_all, u0 + stop - unit);
        unit += u1 - u0;
        // (the CTA with a stream's first unit says where its parts are, for the merge)
        if (u0 == 0 && threadIdx.x == 0) {
            const long long units = (long long)per_head * p.heads_all, share = min((long long)p.ctas, units), at = (long long)hy * per_head + r;
            p.shared_by[(size_t)block * p.heads_all + hy] = make_int2(blockIdx.x, (int)(((at + u_all) * share - 1) / units) - (int)blockIdx.x + 1);
        }
    } else {
        ++unit;
        u_all = pa_units(p, KEYS, block);
        const int each = (u_all + ranks - 1) / ranks;
        u0 = rank * each;
        u1 = min(u_all, u0 + each);
    }
    finished = u0 == 0 && u1 == u_all;
    req = block;
    int row0 = block, rows = 1;
    if (p.blocks) { req = p.blocks[3 * block]; row0 = p.blocks[3 * block + 1]; rows = p.blocks[3 * block + 2]; }
    pos_last = p.positions[row0 + rows - 1];
    list = p.list ? p.list + ((size_t)block * p.nkv + hy / p.head_blocks) * p.top : nullptr;
    const PaChunks all = pa_chunks(p, KEYS, row0, rows);
    chunk0 = all.first; begin = u0 * PA_WARPS + warp; end = min(all.count, u1 * PA_WARPS);
    turns = begin < end ? (end - begin + PA_WARPS - 1) / PA_WARPS : 0;
    };

    // ---- copies: a lane looks up the page of one of the warp's next 32 turns
    unsigned char* ring = smem + (size_t)warp * PA_STAGES * BYTES;
    const unsigned char* from = nullptr;
    int base = 0;
    auto look_up = [&](int turn) {                     // for turns turn .. turn + 31, a lane one
        const int c = begin + (turn + lane) * PA_WARPS;
        from = nullptr;
        if (c >= end) return;
        int index;
        if (list) {
            index = list[c / per_page];
            base = index * p.page_size + c % per_page * KEYS;
        } else {
            base = (chunk0 + c) * KEYS;
            index = base / p.page_size;
        }
        if (index < 0 || base > pos_last) return;
        const int page = index < p.max_pages && req >= 0 && req < p.n_req ? p.table[(size_t)req * p.max_pages + index] : -1;
        if (page < 0 || page >= p.num_pages) {
            if (p.status) atomicOr(p.status, BG_STATUS_BAD_PAGE);
            return;
        }
        from = p.pool + ((size_t)page * p.nkv + hy / p.head_blocks) * p.block_bytes + (size_t)(base % p.page_size / PK_TILE) * L::TILE;
    };
    auto issue = [&](int turn, int stage) {
        const unsigned long long src = __shfl_sync(0xffffffffu, (unsigned long long)from, turn & 31);
        const int at = __shfl_sync(0xffffffffu, base, turn & 31);
        if (lane == 0) {
            where[warp][stage] = src ? at : -1;
            if (src) {
                mbar_expect_tx(&bars[warp][stage], BYTES);
                pa_bulk_load(ring + stage * BYTES, reinterpret_cast<const unsigned char*>(src), BYTES, &bars[warp][stage]);
            } else {
                mbar_arrive(&bars[warp][stage]);
            }
        }
    };
    int stage = 0;
    unsigned phase = 0;
    bool fine = true;                                  // no wait of this warp has run out
    auto first_copies = [&]() {
        if (turns > 0) look_up(0);
#pragma unroll
        for (int i = 0; i < PA_STAGES; ++i)
            if (i < turns) issue(i, stage + i < PA_STAGES ? stage + i : stage + i - PA_STAGES);
    };
    if (unit >= stop) return;
    next_stream();
    first_copies();
    for (;;) {
    const int kvh = hy / p.head_blocks, head0 = hy % p.head_blocks * p.heads_each, heads = min(p.heads_each, p.group - head0);
    const int row0 = p.blocks ? p.blocks[3 * block + 1] : block, cols = min((p.blocks ? p.blocks[3 * block + 2] : 1) * heads, COLS), pos_first = p.positions[row0];
    const bool whole = finished;
    const size_t slot = ((size_t)blockIdx.x * 2 + (u0 == 0)) * COLS;     // (a run's first stream may have begun before it, its last one may go on behind it)

    // ---- queries: column g of every block of 8, features 64 group + 16 t .. + 15 as four steps of a product
    // (those that meet codes at bits 4 are a 16th)
    unsigned qf[PARTS][NT][GROUPS][8];
    unsigned qsum[NT];                                 // of column g of every block: the sums of its groups, the t-th of three parts
    float mult[NT][2];                                 // of columns 2t, 2t + 1: what their scores are multiplied with
    int seen[NT][2];                                   // the positions of their rows
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int col = nt * 8 + g;
        const bool have = col < cols;
        const int r = have ? col / heads : 0, h = head0 + (have ? col - r * heads : 0);
        const TQ* q = reinterpret_cast<const TQ*>(p.q) + (size_t)(row0 + r) * p.q_stride + (size_t)(kvh * p.group + h) * HD + 16 * t;
        float v[GROUPS][16], top = 0.0f;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
                float e[8] = {};
                if (have) load8(q + gr * PK_GROUP + i, e);
#pragma unroll
                for (int j = 0; j < 8; ++j) { v[gr][i + j] = e[j]; top = fmaxf(top, fabsf(e[j])); }
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int high = max(-20, (int)(__float_as_uint(top) >> 23) - 127);
        const float up = __uint_as_float((unsigned)(227 - high) << 23);          // 2^(100 - high)
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float by = i % 2 ? up * 0.0625f : up;
                float a = v[gr][2 * i] * by, b = v[gr][2 * i + 1] * by;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const __nv_bfloat16 x = __float2bfloat16_rn(a), y = __float2bfloat16_rn(b);
                    qf[part][nt][gr][i] = (unsigned)__bfloat16_as_ushort(x) | (unsigned)__bfloat16_as_ushort(y) << 16;
                    a -= __bfloat162float(x); b -= __bfloat162float(y);
                }
            }
        // the sums as the codes 1 give them, in units of 2^-133 (a column's sum is with the lanes 4 x + column / 2); they go back as the right operand of a
        // product with the pairs' lowest values, k = 2t, 2t + 1 the t-th parts of both groups
        float sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
            float c[4] = {};
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int k = 0; k < 4; ++k) pa_mma(c, PA_ONE, PA_ONE, PA_ONE << 4, PA_ONE << 4, qf[part][nt][gr][2 * k], qf[part][nt][gr][2 * k + 1]);
            const float even = __shfl_sync(0xffffffffu, c[0], g / 2), odd = __shfl_sync(0xffffffffu, c[1], g / 2);
            sums[gr] = g % 2 ? odd : even;
        }
        qsum[nt] = 0;
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            const __nv_bfloat16 x = __float2bfloat16_rn(sums[0]), y = __float2bfloat16_rn(sums[1]);
            if (part == t) qsum[nt] = (unsigned)__bfloat16_as_ushort(x) | (unsigned)__bfloat16_as_ushort(y) << 16;
            sums[0] -= __bfloat162float(x); sums[1] -= __bfloat162float(y);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int mine = nt * 8 + 2 * t + j;
            seen[nt][j] = mine < cols ? p.positions[row0 + mine / heads] : pos_last;
            // back from 2^(100 - high) and the codes' 2^-133 to q . k, times what makes it an exponent of two (or, squashed, a part of the bound)
            const int back = min(33 + __shfl_sync(0xffffffffu, high, (2 * t + j) * 4), 127);
            mult[nt][j] = __uint_as_float((unsigned)(127 + back) << 23) * (p.cap_log2 > 0.0f ? p.scale_over_cap : p.scale_log2);
        }
    }

    const bool capped = p.cap_log2 > 0.0f;
    float o[GROUPS * 4][NT][4] = {}, low[NT][GROUPS][2] = {}, m[NT][2], l[NT][2] = {};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY;

    auto chunk = [&](const unsigned char* stage, int at, auto edge_) {
        constexpr bool EDGE = decltype(edge_)::value;
        float x[CT][NT][4];
        unsigned hidden = 0;                           // EDGE: the numbers of x that their column does not see
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const unsigned char* tile = stage + i * L::TILE;
            unsigned kw[2][GROUPS * 2], kp[2][GROUPS];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const unsigned char* row = tile + (g + 8 * half) * (HD / 2) + t * GROUPS * 8;
                const unsigned char* pair = tile + L::PAIRS + (g + 8 * half) * (2 * GROUPS * 4);
                if constexpr (GROUPS == 2) {
                    const uint4 w = *reinterpret_cast<const uint4*>(row);
                    kw[half][0] = w.x; kw[half][1] = w.y; kw[half][2] = w.z; kw[half][3] = w.w;
                    const uint2 v = *reinterpret_cast<const uint2*>(pair);
                    kp[half][0] = v.x; kp[half][1] = v.y;
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(row);
                    kw[half][0] = w.x; kw[half][1] = w.y;
                    kp[half][0] = *reinterpret_cast<const unsigned*>(pair);
                }
            }
            // lowest (sum q) of both groups at once
            float s[NT][4] = {};
            const unsigned low0 = __byte_perm(kp[0][0], kp[0][GROUPS - 1], 0x7632), low1 = __byte_perm(kp[1][0], kp[1][GROUPS - 1], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) pa_mma(s[nt], low0, low1, 0u, 0u, qsum[nt], 0u);
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
                float c[NT][4] = {};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const unsigned w0 = kw[0][gr * 2 + k / 2], w1 = kw[1][gr * 2 + k / 2];
                    const int n = k % 2 * 2;
                    const unsigned a0 = pa_codes(w0, n), a1 = pa_codes(w1, n), a2 = pa_codes(w0, n + 1), a3 = pa_codes(w1, n + 1);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int part = PARTS - 1; part >= 0; --part) pa_mma(c[nt], a0, a1, a2, a3, qf[part][nt][gr][2 * k], qf[part][nt][gr][2 * k + 1]);
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float step = pair_step(kp[half][gr]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) s[nt][2 * half + j] = fmaf(step, c[nt][2 * half + j], s[nt][2 * half + j]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[i][nt][e] = s[nt][e];
                    if constexpr (EDGE) {
                        const int pos = at + i * PK_TILE + g + (e & 2) * 4, last = seen[nt][e & 1];
                        if (pos > last || (p.window > 0 && pos <= last - p.window)) {
                            x[i][nt][e] = -INFINITY;
                            hidden |= 1u << ((i * NT + nt) * 4 + e);
                        }
                    }
                }
        }
        if (capped) {
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(EDGE && (hidden >> ((i * NT + nt) * 4 + e) & 1))) x[i][nt][e] = pa_squashed<F32>(x[i][nt][e] * mult[nt][e & 1], p.cap_log2);
        }
        // The reference maximum of a column moves when some lane has a score 2^8 above it (all lanes of a column have to have the same one, and finding the
        // largest costs three exchanges): until then weights up to 2^8 are as good as those up to 1.
        float top[NT][2];
        bool grew = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float v = x[0][nt][j];
#pragma unroll
                for (int i = 0; i < CT; ++i) v = fmaxf(v, fmaxf(x[i][nt][j], x[i][nt][j + 2]));
                top[nt][j] = capped ? v : v * mult[nt][j];
                grew |= top[nt][j] > m[nt][j] + PA_SLACK;
            }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float v = top[nt][j];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
                    v = fmaxf(m[nt][j], v);
                    const float keep = v == m[nt][j] ? 1.0f : F32 ? exp2f(m[nt][j] - v) : pa_exp2(m[nt][j] - v);
                    m[nt][j] = v;
                    l[nt][j] *= keep;
#pragma unroll
                    for (int gr = 0; gr < GROUPS; ++gr) low[nt][gr][j] *= keep;
#pragma unroll
                    for (int i = 0; i < GROUPS * 4; ++i) { o[i][nt][j] *= keep; o[i][nt][j + 2] *= keep; }
                }
        }
        float less[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) less[nt][j] = (F32 ? 0.0f : PA_UP) - (m[nt][j] == -INFINITY ? 0.0f : m[nt][j]);
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const unsigned char* tile = stage + i * L::TILE;
            float w[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = fmaf(x[i][nt][e], capped ? 1.0f : mult[nt][e & 1], less[nt][e & 1]);
                    w[nt][e] = F32 ? exp2f(z) * 0x1p64f : pa_exp2(z);    // (a float next to PA_UP has 6 bits fewer behind its point)
                    l[nt][e & 1] += w[nt][e];
                }
            unsigned vw[GROUPS][4], vp[2][GROUPS];     // words of positions 2t, 2t + 1, 2t + 8, 2t + 9; pairs of positions g, g + 8
            if constexpr (GROUPS == 2) {
                const uint4 a = *reinterpret_cast<const uint4*>(tile + L::CODES + lane * 16), b = *reinterpret_cast<const uint4*>(tile + L::CODES + 512 + lane * 16);
                vw[0][0] = a.x; vw[1][0] = a.y; vw[0][1] = a.z; vw[1][1] = a.w;
                vw[0][2] = b.x; vw[1][2] = b.y; vw[0][3] = b.z; vw[1][3] = b.w;
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(tile + L::CODES + lane * 16);
                vw[0][0] = a.x; vw[0][1] = a.y; vw[0][2] = a.z; vw[0][3] = a.w;
            }
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int gr = 0; gr < GROUPS; ++gr)
                    vp[half][gr] = *reinterpret_cast<const unsigned*>(tile + L::PAIRS + (g + 8 * half) * (2 * GROUPS * 4) + (GROUPS + gr) * 4);
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
                unsigned b[PARTS][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float step = pair_step(vp[half][gr]), lowest = F32 ? pair_lowest(vp[half][gr]) : fmaf(8.0f, step, pair_lowest(vp[half][gr]));
                        float e[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float weight = w[nt][2 * half + j];
                            e[j] = weight * step;
                            float add = weight * lowest;
                            if constexpr (EDGE) {      // (what lies in a place that is not seen may be no number)
                                if (hidden >> ((i * NT + nt) * 4 + 2 * half + j) & 1) e[j] = add = 0.0f;
                            }
                            low[nt][gr][j] += add;
                        }
                        if constexpr (F32) {
#pragma unroll
                            for (int part = 0; part < PARTS; ++part) {
                                const __nv_bfloat16 a = __float2bfloat16_rn(e[0]), c = __float2bfloat16_rn(e[1]);
                                b[part][nt][half] = pa_transposed((unsigned)__bfloat16_as_ushort(a) | (unsigned)__bfloat16_as_ushort(c) << 16);
                                e[0] -= __bfloat162float(a); e[1] -= __bfloat162float(c);
                            }
                        } else {
                            b[0][nt][half] = pa_transposed(pa_pack(e[0], e[1]));
                        }
                    }
                if constexpr (!F32) {                  // less 8 (p step) as it was rounded; an eighth of it in each of the 8 lanes whose sums meet
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float sum[4] = {low[nt][gr][0], low[nt][gr][1], 0.0f, 0.0f};
                        pa_mma(sum, PA_MINUS, PA_MINUS, PA_MINUS, PA_MINUS, b[0][nt][0], b[0][nt][1]);
                        low[nt][gr][0] = sum[0]; low[nt][gr][1] = sum[1];
                    }
                }
                const unsigned ab[2] = {__byte_perm(vw[gr][0], vw[gr][1], 0x5410), __byte_perm(vw[gr][0], vw[gr][1], 0x7632)};
                const unsigned cd[2] = {__byte_perm(vw[gr][2], vw[gr][3], 0x5410), __byte_perm(vw[gr][2], vw[gr][3], 0x7632)};
#pragma unroll
                for (int k = 0; k < 4; ++k) {          // features 8 g + 2 k (rows g of the product) and 8 g + 2 k + 1 (rows g + 8)
                    const int n = k % 2 * 2;
                    const unsigned a0 = pa_codes(ab[k / 2], n), a1 = pa_codes(ab[k / 2], n + 1);
                    const unsigned a2 = pa_codes(cd[k / 2], n), a3 = pa_codes(cd[k / 2], n + 1);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if constexpr (F32) {           // (the tensor cores' sums are cut off, not rounded: over many positions that shows, so only a tile's are theirs)
                            float sum[4] = {};
#pragma unroll
                            for (int part = PARTS - 1; part >= 0; --part) pa_mma(sum, a0, a1, a2, a3, b[part][nt][0], b[part][nt][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[gr * 4 + k][nt][e] += sum[e];
                        } else {
                            pa_mma(o[gr * 4 + k][nt], a0, a1, a2, a3, b[0][nt][0], b[0][nt][1]);
                        }
                    }
                }
            }
        }
    };

    int turn = 0;
    for (; fine && turn < turns; ++turn) {
        fine = __all_sync(0xffffffffu, mbar_wait(&bars[warp][stage], phase, &gave_up));
        if (!fine) break;                              // (turn stays)
        const int at = where[warp][stage];
        if (at >= 0) {
            if (at + KEYS - 1 > pos_first || (p.window > 0 && at <= pos_last - p.window)) chunk(ring + stage * BYTES, at, std::true_type{});
            else chunk(ring + stage * BYTES, at, std::false_type{});
        }
        __syncwarp();
        const int next = turn + PA_STAGES;
        if (next < turns) {
            if ((next & 31) == 0) look_up(next);
            issue(next, stage);
        }
        if (++stage == PA_STAGES) { stage = 0; phase ^= 1u; }
    }
    if (!fine && turn < turns) {
        // a copy did not come: those of this warp that are on their way are waited for, and the status says so; the warp asks for no more (its results
        // still meet the others', so that nobody waits for it)
        if (lane == 0 && p.status) atomicOr(p.status, BG_STATUS_TIMEOUT);
        for (int i = turn; i < min(turns, turn + PA_STAGES); ++i) {
            mbar_wait(&bars[warp][stage], phase);
            if (++stage == PA_STAGES) { stage = 0; phase ^= 1u; }
        }
    }

    // ---- the next stream's copies come while this one's results meet
    const bool more = SHARE && unit < stop;
    if (more) {
        next_stream();
        if (fine) first_copies();
        else turns = 0;
    }

    // ---- the warps' results meet
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
#pragma unroll
                for (int gr = 0; gr < GROUPS; ++gr) low[nt][gr][j] += __shfl_xor_sync(0xffffffffu, low[nt][gr][j], d);
            }
    __syncthreads();                                   // (the stream before this one is read out)
    float* res = reinterpret_cast<float*>(smem + (size_t)PA_WARPS * PA_STAGES * BYTES);
    float2* ml = reinterpret_cast<float2*>(res + PA_WARPS * COLS * S::ROW);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = nt * 8 + 2 * t + j;
            if (g == 0) ml[warp * COLS + col] = make_float2(m[nt][j], l[nt][j]);
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
                const float add = low[nt][gr][j], even = 0x1p100f, odd = 0x1p96f;        // (back from 2^-133, and from 16 times that)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<float2*>(res + (size_t)(warp * COLS + col) * S::ROW + gr * PK_GROUP + 8 * g + 2 * k) =
                        make_float2(fmaf(o[gr * 4 + k][nt][j] * even, 0x1p33f, add), fmaf(o[gr * 4 + k][nt][j + 2] * odd, 0x1p33f, add));
            }
        }
    __syncthreads();
    auto write = [&](int col, int f, float2 v, float top, float sum) {         // a finished pair of features
        const int r = col / heads, h = kvh * p.group + head0 + col - r * heads;
        float by = 1.0f;
        if (p.sink) {
            const float at = (p.sink_w ? p.sink_w[h] : 0.0f) * PA_LOG2E, most = fmaxf(top, at);
            by = top == -INFINITY ? (sum == 0.0f ? 0.0f : 1.0f) : exp2f(top - most);
            sum = fmaf(sum, by, exp2f(at - most) * 0x1p64f);         // (as the weights)
        }
        by = sum == 0.0f ? 0.0f : by / sum;            // (a row that sees nothing is nought)
        TQ* out = reinterpret_cast<TQ*>(p.out) + (size_t)(row0 + r) * p.out_stride + (size_t)h * HD + f;
        if constexpr (F32) *reinterpret_cast<float2*>(out) = make_float2(v.x * by, v.y * by);
        else *reinterpret_cast<__nv_bfloat162*>(out) = __floats2bfloat162_rn(v.x * by, v.y * by);
    };
    for (int i = threadIdx.x; i < cols * (HD / 2); i += PA_THREADS) {
        const int col = i / (HD / 2), f = i % (HD / 2) * 2;
        float2 each[PA_WARPS];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) { each[w] = ml[w * COLS + col]; top = fmaxf(top, each[w].x); }
        const float from = top == -INFINITY ? 0.0f : top;
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) {
            const float by = exp2f(each[w].x - from);  // (nothing seen: 0)
            const float2 a = *reinterpret_cast<const float2*>(res + (size_t)(w * COLS + col) * S::ROW + f);
            // (scores that are no numbers have no maximum: they show by their sum)
            sum = fmaf(each[w].y, each[w].x == -INFINITY ? 1.0f : by, sum);
            v.x = fmaf(a.x, by, v.x); v.y = fmaf(a.y, by, v.y);
        }
        if (ranks > 1) {                               // to the CTA that joins this column
            const unsigned at = peer_addr(smem_u32(before), (unsigned)(col % ranks)) + 4u * (unsigned)((rank * ((COLS + ranks - 1) / ranks) + col / ranks) * (HD + 2));
            st_cluster(at + 4 * f, v.x); st_cluster(at + 4 * f + 4, v.y);
            if (f == 0) { st_cluster(at + 4 * HD, top); st_cluster(at + 4 * HD + 4, sum); }
            continue;
        }
        if (SHARE && !whole) {
            reinterpret_cast<float2*>(p.part_o + (slot + col) * HD)[i % (HD / 2)] = v;
            if (f == 0) reinterpret_cast<float2*>(p.part_ml)[slot + col] = make_float2(top, sum);
            continue;
        }
        write(col, f, v, top, sum);
    }
    if (ranks > 1) {
        cluster_sync_all();
        const int mine = rank < cols ? (cols - rank + ranks - 1) / ranks : 0, apart = (COLS + ranks - 1) / ranks * (HD + 2);
        for (int i = threadIdx.x; i < mine * (HD / 2); i += PA_THREADS) {
            const int f = i % (HD / 2) * 2;
            const float* at = reinterpret_cast<const float*>(before) + i / (HD / 2) * (HD + 2);
            float top = -INFINITY, sum = 0.0f;
            for (int c = 0; c < ranks; ++c) top = fmaxf(top, at[c * apart + HD]);
            const float from = top == -INFINITY ? 0.0f : top;
            float2 v = make_float2(0.0f, 0.0f);
            for (int c = 0; c < ranks; ++c) {
                const float m_c = at[c * apart + HD], by = exp2f(m_c - from);
                const float2 a = *reinterpret_cast<const float2*>(at + c * apart + f);
                sum = fmaf(at[c * apart + HD + 1], m_c == -INFINITY ? 1.0f : by, sum);
                v.x = fmaf(a.x, by, v.x); v.y = fmaf(a.y, by, v.y);
            }
            write(rank + i / (HD / 2) * ranks, f, v, top, sum);
        }
    }
    if (!more) break;
    }
}

// out = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m) over the CTAs that share a stream (a stream that one CTA had is done); EACH warps take every EACH-th of
// them and join in their order.
constexpr int PM_WARPS = 8;
template <int HD, bool F32, int EACH>
__global__ void __launch_bounds__(PM_WARPS * 32) packed_merge_kernel(const PaParams p, int cols_most) {
    constexpr int PER = HD / 32, AT_ONCE = 8;
    using TQ = typename std::conditional<F32, float, __nv_bfloat16>::type;
    __shared__ float acc_s[PM_WARPS][HD];
    __shared__ float2 ml_s[PM_WARPS];
    pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % EACH;
    const int block = blockIdx.x, hy = blockIdx.y, kvh = hy / p.head_blocks, head0 = hy % p.head_blocks * p.heads_each, heads = min(p.heads_each, p.group - head0);
    const int col = blockIdx.z * (PM_WARPS / EACH) + warp / EACH;
    pdl_wait();
    const int2 by_ = p.shared_by[(size_t)block * p.heads_all + hy];
    const int first = by_.x, parts = by_.y;
    if (parts == 1) return;
    int row0 = block, rows = 1;
    if (p.blocks) { row0 = p.blocks[3 * block + 1]; rows = p.blocks[3 * block + 2]; }
    const bool idle = col >= rows * heads || col >= cols_most;
    // the first CTA has its part in its second place, the others theirs in their first
    auto place = [&](int i) { return ((size_t)(first + i) * 2 + (i == 0)) * cols_most + (idle ? 0 : col); };
    float m = -INFINITY, l = 0.0f, acc[PER] = {};
    for (int i0 = part; !idle && i0 < parts; i0 += AT_ONCE * EACH) {
        float2 ml[AT_ONCE];
        float v[AT_ONCE][PER];
        float top = m;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int i = i0 + j * EACH;
            const bool have = i < parts;
            const size_t from = place(have ? i : 0);
            ml[j] = have ? reinterpret_cast<const float2*>(p.part_ml)[from] : make_float2(-INFINITY, 0.0f);
            if constexpr (PER == 4) {
                const float4 a = have ? *reinterpret_cast<const float4*>(p.part_o + from * HD + lane * PER) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                v[j][0] = a.x; v[j][1] = a.y; v[j][2] = a.z; v[j][3] = a.w;
            } else {
                const float2 a = have ? *reinterpret_cast<const float2*>(p.part_o + from * HD + lane * PER) : make_float2(0.0f, 0.0f);
                v[j][0] = a.x; v[j][1] = a.y;
            }
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) top = fmaxf(top, ml[j].x);
        const float from = top == -INFINITY ? 0.0f : top, keep = m == -INFINITY ? 1.0f : exp2f(m - from);
        l *= keep;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] *= keep;
        m = top;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const float by = ml[j].x == -INFINITY ? 1.0f : exp2f(ml[j].x - from);      // (scores that are no numbers have no maximum)
            l = fmaf(ml[j].y, by, l);
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] = fmaf(v[j][e], by, acc[e]);
        }
    }
    if constexpr (EACH > 1) {
#pragma unroll
        for (int e = 0; e < PER; ++e) acc_s[warp][lane * PER + e] = acc[e];
        if (lane == 0) ml_s[warp] = make_float2(m, l);
        __syncthreads();
        if (part) return;
        float top = m;
#pragma unroll
        for (int j = 1; j < EACH; ++j) top = fmaxf(top, ml_s[warp + j].x);
        const float from = top == -INFINITY ? 0.0f : top, keep = m == -INFINITY ? 1.0f : exp2f(m - from);
        l *= keep;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] *= keep;
        m = top;
#pragma unroll
        for (int j = 1; j < EACH; ++j) {
            const float2 ml = ml_s[warp + j];
            const float by = ml.x == -INFINITY ? 1.0f : exp2f(ml.x - from);
            l = fmaf(ml.y, by, l);
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] = fmaf(acc_s[warp + j][lane * PER + e], by, acc[e]);
        }
    }
    if (idle) return;
    const int r = col / heads, h = kvh * p.group + head0 + col - r * heads;
    float by = 1.0f;
    if (p.sink) {
        const float at = (p.sink_w ? p.sink_w[h] : 0.0f) * PA_LOG2E, most = fmaxf(m, at);
        by = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - most);
        l = fmaf(l, by, exp2f(at - most) * 0x1p64f);
    }
    by = l == 0.0f ? 0.0f : by / l;
    TQ* out = reinterpret_cast<TQ*>(p.out) + (size_t)(row0 + r) * p.out_stride + (size_t)h * HD + lane * PER;
#pragma unroll
    for (int e = 0; e < PER; e += 2) {
        if constexpr (F32) *reinterpret_cast<float2*>(out + e) = make_float2(acc[e] * by, acc[e + 1] * by);
        else *reinterpret_cast<__nv_bfloat162*>(out + e) = __floats2bfloat162_rn(acc[e] * by, acc[e + 1] * by);
    }
}

template <int HD, int NT, bool F32, int CT>
static int pa_launch(const PaParams& p, int n, cudaStream_t stream) {
    const size_t smem = (size_t)PA_WARPS * PA_STAGES * CT * Packed<HD>::TILE + PaShape<HD, NT, F32>::JOIN;      // the rings, and where results meet
    if (!p.ctas) {
        cudaError_t e = smem_limit(packed_attention_kernel<HD, NT, F32, CT, false>, smem);
        if (e != cudaSuccess) return (int)e;
        e = launch_cluster(packed_attention_kernel<HD, NT, F32, CT, false>, dim3(n, p.heads_all, p.cluster), dim3(PA_THREADS), smem, stream, p.cluster, p);
        return e == cudaSuccess ? BG_OK : (int)e;
    }
    cudaError_t e = smem_limit(packed_attention_kernel<HD, NT, F32, CT, true>, smem);
    if (e != cudaSuccess) return (int)e;
    e = launch(packed_attention_kernel<HD, NT, F32, CT, true>, dim3(p.ctas), dim3(PA_THREADS), smem, stream, p);
    if (e != cudaSuccess) return (int)e;
    constexpr int COLS = 8 * NT;
    // (many CTAs a stream: a CTA joins one column, not a warp: 1 row of 131,072 positions, 4 kv heads, 25.5 us with attention, by warps 32.4; 4 rows 68.5 and
    // 70.2; but 16 rows of 8,000 28.9 and 27.9, 64 rows 76.4 and 72.2)
    e = p.ctas > 8 * n * p.heads_all ? launch(packed_merge_kernel<HD, F32, PM_WARPS>, dim3(n, p.heads_all, COLS), dim3(PM_WARPS * 32), 0, stream, p, COLS)
                                     : launch(packed_merge_kernel<HD, F32, 1>, dim3(n, p.heads_all, NT), dim3(PM_WARPS * 32), 0, stream, p, COLS);
    return e == cudaSuccess ? BG_OK : (int)e;
}

template <int HD, bool F32>
static int pa_sized(const PaParams& p, int n, int nt, cudaStream_t stream) {
    const bool wide = p.page_size % (2 * PK_TILE) == 0;
    if (nt == 1) return wide ? pa_launch<HD, 1, F32, 2>(p, n, stream) : pa_launch<HD, 1, F32, 1>(p, n, stream);
    if constexpr (F32) return BG_ERR_UNSUPPORTED;
    else return wide ? pa_launch<HD, 2, F32, 2>(p, n, stream) : pa_launch<HD, 2, F32, 1>(p, n, stream);
}

}  // namespace bg

using namespace bg;

// Columns of a block of `rows` rows: blocks of 8 (row, head) pairs that one CTA takes (1 or 2; float queries, whose parts fill the registers, 1), and query
// heads of a block.  heads_each * rows fits the columns.
extern "C" int bg_packed_attention_columns(int group, int f32, int rows, int* heads_each) {
    const int most = f32 ? 8 : 16;
    if (group <= 0 || rows <= 0) return BG_ERR_SHAPE;
    *heads_each = group <= most ? group : most;
    if (*heads_each * rows > most) return BG_ERR_UNSUPPORTED;
    return *heads_each * rows <= 8 ? 1 : 2;
}

// The most blocks whose positions CTAs share.
extern "C" int bg_packed_attention_blocks() { return PA_BLOCKS; }

extern "C" int bg_packed_attention_bytes() { return (int)sizeof(PaCall); }

// part_o holds 2 * ctas * columns results, part_ml their maxima and sums and, behind them, two whole numbers for every stream.
extern "C" int bg_packed_attention(const void* call, cudaStream_t stream) {
    const PaCall& c = *(const PaCall*)call;
    if (c.hd != 64 && c.hd != 128) return BG_ERR_UNSUPPORTED;
    if (c.n <= 0) return BG_OK;
    if (c.page_size <= 0 || c.page_size % PK_TILE || c.nkv <= 0 || c.nh <= 0 || c.nh % c.nkv || c.ctas < 0 || c.cluster < 1 || c.cluster > 8 || c.num_pages <= 0 || c.max_pages <= 0
        || c.window < 0 || !(c.scale > 0.0f)) return BG_ERR_SHAPE;
    if (c.block_bytes % 16 || c.block_bytes < c.page_size / PK_TILE * packed_tile_bytes(c.hd) || (c.ctas && c.n > PA_BLOCKS)
        || (c.list && (c.top <= 0 || c.rows != 1))) return BG_ERR_SHAPE;
    if (c.dtype != BG_DTYPE_F32 && c.dtype != BG_DTYPE_BF16) return BG_ERR_DTYPE;
    const bool f32 = c.dtype == BG_DTYPE_F32;
    const long long size = f32 ? 4 : 2;
    if ((uintptr_t)c.pool % 16 || ((long long)(uintptr_t)c.q | c.q_stride * size) % 16 || ((long long)(uintptr_t)c.out | c.out_stride * size) % (2 * size)) return BG_ERR_ALIGN;
    if ((c.ctas > 0) != (c.part_o != nullptr) || (c.part_o == nullptr) != (c.part_ml == nullptr) || (uintptr_t)c.part_o % 16 || (uintptr_t)c.part_ml % 8) return BG_ERR_SHAPE;
    PaParams p;
    static_cast<PaCall&>(p) = c;
    const int nt = bg_packed_attention_columns(c.nh / c.nkv, f32, c.rows, &p.heads_each);
    if (nt < 0) return nt;
    p.group = c.nh / c.nkv;
    p.head_blocks = (p.group + p.heads_each - 1) / p.heads_each;
    if ((long long)c.nkv * p.head_blocks > 65535) return BG_ERR_SHAPE;
    p.heads_all = c.nkv * p.head_blocks;
    p.shared_by = reinterpret_cast<int2*>(c.part_ml + (size_t)4 * c.ctas * 8 * nt);
    p.scale_log2 = c.scale * PA_LOG2E;
    p.cap_log2 = c.softcap > 0.0f ? c.softcap * PA_LOG2E : 0.0f;
    p.scale_over_cap = c.softcap > 0.0f ? c.scale / c.softcap : 0.0f;
    if (c.hd == 64) return f32 ? pa_sized<64, true>(p, c.n, nt, stream) : pa_sized<64, false>(p, c.n, nt, stream);
    return f32 ? pa_sized<128, true>(p, c.n, nt, stream) : pa_sized<128, false>(p, c.n, nt, stream);
}
