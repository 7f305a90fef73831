// Writing and reading pages that hold keys and values in 4 bits (packed.cuh says how): the append of a step's rows with the rotation of queries and keys on
// the way, rows read back, the smallest and largest values of a filled page's keys, and pages written out in half precision for the
// prompt attention.
//
// A group of 64 features x becomes  lowest = bf16(min x),  step = bf16((max x - lowest) / 15),  u = clamp(round((x - lowest) / step), 0, 15), nought where the step
// is not positive.  The pair is rounded before the codes are made, so that they are the nearest ones to what is read back: a value is off by half a step, or by
// as much as rounding moved the end of the range that it lies beyond, which is up to 2^-8 of lowest below and 2^-8 of 15 steps above.  So a group needs a range that is
// not small beside its values: one of 100.30 .. 100.45 has lowest 100.5, a step below nought and every code 0, 0.2 off.  x is the rotated key in float, never
// rounded to bfloat16.  A group with a value that is not finite, or whose range is
// not, is not a number throughout, as attention over it would be.  No result hangs on which thread wrote first: a position has one writer.
#include <cuda_fp16.h>

#include "packed.cuh"

namespace bg {

// ------------------------------------------------------------------------------------------------ append
// (the host side packs this and the other calls' fields in their order)
struct PkAppend {
    const void* src; long long src_stride, part_stride;
    void* q_out; long long q_stride;
    const float* cos_sin;
    const int* positions; const int* row_req; const int* block_table;
    unsigned char* pool; long long block_bytes;
    unsigned* status;
    int src_dtype, q_dtype, parts, max_pages, num_pages, page_size, T, n_req, nh, nkv, hd, rot, interleaved, pad;
};

// Eight neighbouring features of a row (summed over partial results).
template <typename T>
__device__ __forceinline__ void load8_parts(const T* p, int parts, long long stride, float (&v)[8]) {
    load8(p, v);
    for (int i = 1; i < parts; ++i) {
        float w[8];
        load8(p + i * stride, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += w[j];
    }
}
// The (cos, sin) of features f .. f + 7's rotation and their partners in the row (SPLIT: halves of whole pieces of 8; else anything, neighbours or halves).
template <typename T, bool SPLIT>
__device__ __forceinline__ void rotation8(const PkAppend& p, const T* head, const float2* table, int f, const float (&x)[8], float (&y)[8], float (&cs)[8], float (&sn)[8]) {
    const int half = p.rot / 2;
    if constexpr (SPLIT) {
        const bool front = f < half;
        load8_parts<T>(head + (front ? f + half : f - half), p.parts, p.part_stride, y);
        const float4* from = reinterpret_cast<const float4*>(table + (front ? f : f - half));
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float4 c = from[j / 2];
            cs[j] = c.x; sn[j] = front ? -c.y : c.y; cs[j + 1] = c.z; sn[j + 1] = front ? -c.w : c.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = f + j;
            cs[j] = 1.0f; sn[j] = 0.0f; y[j] = 0.0f;
            if (at >= p.rot) continue;
            const float2 c = table[p.interleaved ? at / 2 : at < half ? at : at - half];
            cs[j] = c.x;
            sn[j] = (p.interleaved ? at % 2 == 0 : at < half) ? -c.y : c.y;              // (a cos - b sin, and b cos + a sin for the partner)
            y[j] = p.interleaved ? x[j ^ 1] : sum_parts(head + (at < half ? at + half : at - half), p.parts, (size_t)p.part_stride);
        }
    }
}

// Queries: HD / 16 lanes take a head of a row, a lane two pieces of 8 features: with SPLIT a piece and its partner, so that each is read once.
constexpr int PK_THREADS = 256;
template <typename TS, typename TQ, int HD, bool SPLIT>
__device__ __forceinline__ void append_query(const PkAppend& p, long long item, int l) {
    const int t = (int)(item / p.nh), h = (int)(item - (long long)t * p.nh);
    const TS* head = reinterpret_cast<const TS*>(p.src) + (size_t)t * p.src_stride + (size_t)h * HD;
    const float2* table = reinterpret_cast<const float2*>(p.cos_sin) + (size_t)t * (p.rot / 2);
    TQ* out = reinterpret_cast<TQ*>(p.q_out) + (size_t)t * p.q_stride + (size_t)h * HD;
    float a[8], b[8];
    if constexpr (SPLIT) {
        const int half = p.rot / 2;
        const bool turned = 8 * l < half;
        const int f = turned ? 8 * l : p.rot + 2 * (8 * l - half), g = turned ? f + half : f + 8;
        load8_parts<TS>(head + f, p.parts, p.part_stride, a);
        load8_parts<TS>(head + g, p.parts, p.part_stride, b);
        if (turned) {
            const float4* from = reinterpret_cast<const float4*>(table + f);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float4 c = from[j / 2];
                const float a0 = a[j], a1 = a[j + 1];
                a[j] = __fadd_rn(__fmul_rn(a0, c.x), -__fmul_rn(b[j], c.y));
                b[j] = __fadd_rn(__fmul_rn(b[j], c.x), __fmul_rn(a0, c.y));
                a[j + 1] = __fadd_rn(__fmul_rn(a1, c.z), -__fmul_rn(b[j + 1], c.w));
                b[j + 1] = __fadd_rn(__fmul_rn(b[j + 1], c.z), __fmul_rn(a1, c.w));
            }
        }
        store8(out + f, a);
        store8(out + g, b);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int f = 16 * l + 8 * i;
            float y[8], cs[8], sn[8];
            load8_parts<TS>(head + f, p.parts, p.part_stride, a);
            if (f < p.rot) {
                rotation8<TS, false>(p, head, table, f, a, y, cs, sn);
#pragma unroll
                for (int j = 0; j < 8; ++j) a[j] = __fadd_rn(__fmul_rn(a[j], cs[j]), __fmul_rn(y[j], sn[j]));
            }
            store8(out + f, a);
        }
    }
}

// Keys and values: HD / 8 lanes take a head of a row, a lane eight neighbouring features, which are a word of codes; a group's 8 lanes find its smallest and
// largest by shuffles.  The codes are those that 64 bits give: everything is done in 32 first, with a bound on how far off that may be, and where the bound
// reaches the border of two codes, or of two roundings of the pair, the warp does its heads again in 64 (two or three warps of a thousand).  What
// is left of x - lowest beside the nearest whole number of steps is one fused multiply-add, exact where that difference is (bfloat16 that was not rotated): a
// comparison with half a step then decides as 64 bits do, without a division.
// The first CTAs take the queries' heads, the others the keys' and values', both row after row: bound by the latency of a CTA (its loads, one behind the
// other), so every lane has work and as many CTAs as can be are under way.  4,917 rows of 36 heads (86 MB): 33 us, 40 % of the bandwidth of a copy; 90 us with a CTA
// for some heads of one row, four features a lane and every head on the keys' path.
template <typename TS, typename TQ, int HD, bool SPLIT>
__global__ void __launch_bounds__(PK_THREADS, 4) packed_append_kernel(const PkAppend p, int other_ctas) {
    constexpr int LANES = HD / 8;
    pdl_launch();
    pdl_wait();
    if ((int)blockIdx.x >= other_ctas) {
        const long long item = (long long)((int)blockIdx.x - other_ctas) * (PK_THREADS / (HD / 16)) + threadIdx.x / (HD / 16);
        if (item < (long long)p.T * p.nh) append_query<TS, TQ, HD, SPLIT>(p, item, threadIdx.x % (HD / 16));
        return;
    }
    const long long item = (long long)blockIdx.x * (PK_THREADS / LANES) + threadIdx.x / LANES;
    const int l = threadIdx.x % LANES, f = l * 8;
    const bool idle = item >= (long long)p.T * 2 * p.nkv;              // (stays for the shuffles)
    const int t = idle ? 0 : (int)(item / (2 * p.nkv)), h = p.nh + (idle ? 0 : (int)(item - (long long)t * 2 * p.nkv));
    const TS* row = reinterpret_cast<const TS*>(p.src) + (size_t)t * p.src_stride + (size_t)h * HD;
    const bool key = h < p.nh + p.nkv;
    // (where the row goes is looked up while its features are on their way)
    const int pos = p.positions[t], req = p.row_req[t];
    float x[8], y[8] = {}, cs[8], sn[8];               // y: a feature's partner
    load8_parts<TS>(row + f, p.parts, p.part_stride, x);
    int page = -1, at = 0;
    if (pos >= 0 && req >= 0 && req < p.n_req) {
        const int index = pos / p.page_size;
        at = pos - index * p.page_size;
        if (index < p.max_pages) page = p.block_table[(size_t)req * p.max_pages + index];
    }
    const bool turned = key && f < p.rot;
    float r[8], off = 0.0f;                            // off: the largest |x cos| + |partner sin|
    if (turned) {
        rotation8<TS, SPLIT>(p, row, reinterpret_cast<const float2*>(p.cos_sin) + (size_t)t * (p.rot / 2), f, x, y, cs, sn);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = __fmul_rn(x[j], cs[j]), b = __fmul_rn(y[j], sn[j]);
            r[j] = __fadd_rn(a, b);
            off = fmaxf(off, fabsf(a) + fabsf(b));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = x[j];
    }
    float lo = r[0], hi = r[0], nought = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) { lo = fminf(lo, r[j]); hi = fmaxf(hi, r[j]); nought = fmaf(0.0f, r[j], nought); }
    int sound = nought == 0.0f;                        // (nought times what is not finite is no number)
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        off = fmaxf(off, __shfl_xor_sync(0xffffffffu, off, o));
        sound &= __shfl_xor_sync(0xffffffffu, sound, o);
    }
    off *= 1.5e-7f;                                    // a rotated feature's error: 2^-24 of each product and of their sum
    __nv_bfloat16 lowest = __float2bfloat16_rn(lo);
    float base = __bfloat162float(lowest);
    const float span = __fmul_rn(__fsub_rn(hi, base), 1.0f / 15.0f), span_off = fmaf(3e-7f, fabsf(span), 0.1f * off);
    sound &= fabsf(span) < INFINITY && fabsf(base) < INFINITY;
    __nv_bfloat16 step = __float2bfloat16_rn(span);
    float s = __bfloat162float(step);
    float by = s > 0.0f ? s : 1.0f;                    // (a group of one value: every code 0)
    int near = __bfloat16_as_ushort(__float2bfloat16_rn(lo - off)) != __bfloat16_as_ushort(__float2bfloat16_rn(lo + off))
            || __bfloat16_as_ushort(__float2bfloat16_rn(span - span_off)) != __bfloat16_as_ushort(__float2bfloat16_rn(span + span_off));
    const float inv = __frcp_rn(by), half_step = 0.5f * by;
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // the whole number next to d / by, by adding 1.5 2^23 (whose last bit is then its parity), and what is left of d, which is exact up to one rounding
        const float d = __fsub_rn(r[j], base), t = fmaf(d, inv, 12582912.0f), k = __fsub_rn(t, 12582912.0f), left = fmaf(-k, by, d);
        const float over = __fsub_rn(fabsf(left), half_step);
        u[j] = over > 0.0f || (over == 0.0f && (__float_as_uint(t) & 1u)) ? k + copysignf(1.0f, left) : k;
        // (the two errors of the difference x - lowest: both nought where it is exact)
        const bool sure = sizeof(TS) == 2 && p.parts == 1 && !turned && __fadd_rn(d, base) == r[j] && __fsub_rn(r[j], d) == base;
        near |= !sure && fabsf(over) <= fmaf(2.5e-7f, fabsf(d) + by, off);
    }
    if (!(by >= 1e-36f)) near = 1;                     // (a step whose reciprocal or borders leave the normal range)
    if (__any_sync(0xffffffffu, near && sound && !idle)) {
        double w[8], least64, most64;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = turned ? (double)x[j] * cs[j] + (double)y[j] * sn[j] : (double)x[j];
            least64 = j ? fmin(least64, w[j]) : w[j];
            most64 = j ? fmax(most64, w[j]) : w[j];
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            least64 = fmin(least64, __shfl_xor_sync(0xffffffffu, least64, o));
            most64 = fmax(most64, __shfl_xor_sync(0xffffffffu, most64, o));
        }
        lowest = __float2bfloat16_rn((float)least64);
        base = __bfloat162float(lowest);
        step = __float2bfloat16_rn((float)((most64 - (double)base) / 15.0));
        s = __bfloat162float(step);
        by = s > 0.0f ? s : 1.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = (float)rint((w[j] - (double)base) / (double)by);
    }
    if (idle) return;
    // four codes to a whole number below 2^16, whose bits 2^23 lays bare (conversions are for units of a quarter of the width)
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = fminf(fmaxf(u[e], 0.0f), 15.0f);
    auto four = [](float a, float b, float c, float d) { return __float_as_uint(fmaf(4096.0f, d, fmaf(256.0f, c, fmaf(16.0f, b, a))) + 8388608.0f); };
    unsigned word = key ? __byte_perm(four(u[0], u[2], u[4], u[6]), four(u[1], u[3], u[5], u[7]), 0x5410)
                        : __byte_perm(four(u[0], u[1], u[2], u[3]), four(u[4], u[5], u[6], u[7]), 0x5410);
    if (!sound) {
        lowest = step = __float2bfloat16_rn(__int_as_float(0x7fffffff));
        word = 0;
    }
    if (page < 0 || page >= p.num_pages) {
        if (p.status && l == 0) atomicOr(p.status, BG_STATUS_BAD_PAGE);
        return;
    }
    const int slot = at % PK_TILE, kvh = h - p.nh - (key ? 0 : p.nkv);
    unsigned char* tile = p.pool + ((size_t)page * p.nkv + kvh) * p.block_bytes + (size_t)(at / PK_TILE) * Packed<HD>::TILE;
    *reinterpret_cast<unsigned*>(tile + (key ? Packed<HD>::key_word(slot, f) : Packed<HD>::value_word(slot, f))) = word;
    if (l % 8 == 0) {
        const unsigned pair = (unsigned)__bfloat16_as_ushort(step) | (unsigned)__bfloat16_as_ushort(lowest) << 16;
        *reinterpret_cast<unsigned*>(tile + Packed<HD>::pair_word(slot, key ? 0 : 1, l / 8)) = pair;
    }
}

// ------------------------------------------------------------------------------------------------ rows read back
struct PkRead {
    unsigned char* pool; long long block_bytes;
    const int* positions; const int* row_req; const int* block_table;
    void* out;
    unsigned* status;
    int out_dtype, max_pages, num_pages, page_size, n_req, T, nkv, hd;
};

// out[t, keys and values, kv head, feature]: a thread reads a word of codes and writes its 8 values.
template <typename TO, int HD>
__global__ void __launch_bounds__(PK_THREADS) packed_rows_kernel(const PkRead p) {
    constexpr int WORDS = HD / 8;
    pdl_launch();
    const int per_row = 2 * p.nkv * WORDS, i = blockIdx.y * PK_THREADS + threadIdx.x, t = blockIdx.x;
    const int value = i / (p.nkv * WORDS), kvh = i / WORDS % p.nkv, f = i % WORDS * 8;
    pdl_wait();                                        // (all warps of a CTA, those without work too)
    if (i >= per_row) return;
    const int pos = p.positions[t], req = p.row_req[t], index = pos / p.page_size;
    const int page = pos >= 0 && req >= 0 && req < p.n_req && index < p.max_pages ? p.block_table[(size_t)req * p.max_pages + index] : -1;
    TO* out = reinterpret_cast<TO*>(p.out) + ((size_t)t * 2 * p.nkv + (size_t)value * p.nkv + kvh) * HD + f;
    float v[8] = {};
    if (page < 0 || page >= p.num_pages) {
        if (p.status) atomicOr(p.status, BG_STATUS_BAD_PAGE);
    } else {
        const int at = pos % p.page_size, slot = at % PK_TILE;
        const unsigned char* tile = p.pool + ((size_t)page * p.nkv + kvh) * p.block_bytes + (size_t)(at / PK_TILE) * Packed<HD>::TILE;
        const unsigned pair = *reinterpret_cast<const unsigned*>(tile + Packed<HD>::pair_word(slot, value, f / PK_GROUP));
        const unsigned word = *reinterpret_cast<const unsigned*>(tile + (value ? Packed<HD>::value_word(slot, f) : Packed<HD>::key_word(slot, f)));
        if (value) packed_values<false>(word, pair, v);
        else packed_values<true>(word, pair, v);
    }
    store8(out, v);
}

// ------------------------------------------------------------------------------------------------ bounds of filled pages
// A row that fills its page (its position is the page's last) has the CTA of its rows find the smallest and largest value of every feature of the page's keys, as
// they are read back, rounded to the nearest bfloat16 number: a feature may lie beyond its bound by up to 2^-8 of itself.  What a page's bounds are hangs on the page alone, whoever wrote it and in how many steps.  A CTA looks at PK_ROWS rows of one kv head; for
// one that fills its page a thread takes a word of 8 features of every (PK_THREADS / words)-th position; a value that is no number stays one.  (A CTA for every
// row: 26 us for 4,917 rows, of CTAs that had nothing to do; a warp for every row: 19 us for the page that one row fills.)
constexpr int PK_ROWS = 8;
__device__ __forceinline__ float least(float a, float b) { return a < b || a != a ? a : b; }
__device__ __forceinline__ float most(float a, float b) { return a > b || a != a ? a : b; }
template <int HD>
__global__ void __launch_bounds__(PK_THREADS) packed_bounds_kernel(const PkRead p) {
    constexpr int WORDS = HD / 8, AT_ONCE = PK_THREADS / WORDS;
    __shared__ float ends[2][AT_ONCE][HD + 1];
    pdl_launch();
    const int kvh = blockIdx.y, row0 = blockIdx.x * PK_ROWS, lane = threadIdx.x % 32;
    pdl_wait();
    const int mine = lane < PK_ROWS && row0 + lane < p.T ? p.positions[row0 + lane] : -1;
    unsigned full = __ballot_sync(0xffffffffu, mine >= 0 && mine % p.page_size == p.page_size - 1);          // (the same in every warp)
    const int w = threadIdx.x % WORDS, first = threadIdx.x / WORDS, f = w * 8;
    for (; full; full &= full - 1) {
        const int t = row0 + __ffs(full) - 1, req = p.row_req[t], index = p.positions[t] / p.page_size;
        const int page = req >= 0 && req < p.n_req && index < p.max_pages ? p.block_table[(size_t)req * p.max_pages + index] : -1;
        if (page < 0 || page >= p.num_pages) {
            if (p.status && threadIdx.x == 0) atomicOr(p.status, BG_STATUS_BAD_PAGE);
            continue;
        }
        unsigned char* block = p.pool + ((size_t)page * p.nkv + kvh) * p.block_bytes;
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
#pragma unroll 4
        for (int at = first; at < p.page_size; at += AT_ONCE) {
            const unsigned char* tile = block + (size_t)(at / PK_TILE) * Packed<HD>::TILE;
            float v[8];
            packed_values<true>(*reinterpret_cast<const unsigned*>(tile + Packed<HD>::key_word(at % PK_TILE, f)),
                                *reinterpret_cast<const unsigned*>(tile + Packed<HD>::pair_word(at % PK_TILE, 0, f / PK_GROUP)), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) { lo[e] = least(v[e], lo[e]); hi[e] = most(v[e], hi[e]); }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) { ends[0][first][f + e] = lo[e]; ends[1][first][f + e] = hi[e]; }
        __syncthreads();
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(block + (size_t)(p.page_size / PK_TILE) * Packed<HD>::TILE);
        for (int i = threadIdx.x; i < 2 * HD; i += PK_THREADS) {
            const int end = i / HD, feature = i % HD;
            float v = ends[end][0][feature];
            for (int j = 1; j < AT_ONCE; ++j) v = end ? most(ends[1][j][feature], v) : least(ends[0][j][feature], v);
            out[i] = __float2bfloat16_rn(v);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ pages in half precision
struct PkUnpack {
    const unsigned char* pool; long long block_bytes;
    const int* positions; const int* block_table;
    const int* longs;                  // [n][3]: request, first row, rows
    const int* ends;                   // [n]: a bound of their positions, or 0: `end` is
    __half* out;                       // [room, 2, nkv, PK_WIDE, HD]
    int* table;                        // [n, table_pages]: their block table
    PkWritten* written;                // [n][nkv]
    unsigned long long* marks;         // [room][nkv][groups]: the page's positions whose values are no numbers, where `written` says that there are some
    int max_pages, num_pages, page_size, n_req, nkv, table_pages, room, end, window;
    unsigned* status;
};
__device__ __forceinline__ int unpack_room(const PkUnpack& p, int n) {
    const int end = p.ends[n];
    return packed_room(p.longs[3 * n + 2], end > 0 ? min(end, p.end) : p.end, p.window);
}

// The page of a tile of 16 positions from `pos0` on that the n-th request's rows read, or -1 (and the status says where a page is not).
__device__ __forceinline__ int unpack_page(const PkUnpack& p, int req, int pos0, int lo, int last, bool say) {
    if (pos0 > last || pos0 + PK_TILE <= lo) return -1;            // (what lies in front of a window may have been given back)
    const int index = pos0 / p.page_size;
    const int page = index < p.max_pages && req >= 0 && req < p.n_req ? p.block_table[(size_t)req * p.max_pages + index] : -1;
    if (page >= 0 && page < p.num_pages) return page;
    if (say && p.status) atomicOr(p.status, BG_STATUS_BAD_PAGE);
    return -1;
}

// How far the keys and the values of each (request, kv head) reach, from their (step, lowest) pairs alone: the power of two that brings the largest between
// 2^14 and 2^15, so that half precision holds them whatever a model's scale is.  A cluster of CTAs takes a request's positions, a thread one at a time, several
// on their way; the CTAs' maxima meet in the first one's shared memory.
constexpr int PK_CLUSTER = 8;
template <int HD>
__global__ void __launch_bounds__(PK_THREADS) packed_reach_kernel(const PkUnpack p) {
    constexpr int GROUPS = Packed<HD>::GROUPS, AT_ONCE = 8;
    __shared__ float every[3][PK_CLUSTER];
    __shared__ float scratch[32];
    pdl_launch();
    const int kvh = blockIdx.x, n = blockIdx.y, rank = blockIdx.z;
    pdl_wait();
    cluster_arrive_relaxed();                          // (the first CTA has begun before its memory is written)
    cluster_wait();
    const int req = p.longs[3 * n], row0 = p.longs[3 * n + 1], rows = p.longs[3 * n + 2];
    const int last = p.positions[row0 + rows - 1], lo = first_visible(p.positions[row0], p.window);
    float top[2] = {0.0f, 0.0f};
    int marked = 0;
    const int stride = PK_CLUSTER * PK_THREADS;
    for (int pos0 = lo / PK_TILE * PK_TILE + rank * PK_THREADS + threadIdx.x; pos0 <= last; pos0 += AT_ONCE * stride) {
        int page[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int pos = pos0 + i * stride;
            page[i] = pos <= last ? unpack_page(p, req, pos / PK_TILE * PK_TILE, lo, last, false) : -1;
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (page[i] < 0) continue;
            const int at = (pos0 + i * stride) % p.page_size;
            const unsigned* pair = reinterpret_cast<const unsigned*>(p.pool + ((size_t)page[i] * p.nkv + kvh) * p.block_bytes + (size_t)(at / PK_TILE) * Packed<HD>::TILE
                                                                     + Packed<HD>::pair_word(at % PK_TILE, 0, 0));
#pragma unroll
            for (int e = 0; e < 2 * GROUPS; ++e) {
                const float lowest = pair_lowest(pair[e]);
                if (!pair_finite(pair[e])) {           // (says nothing of how far the others reach)
                    if (e >= GROUPS) marked |= 1 << (e - GROUPS);
                    continue;
                }
                top[e / GROUPS] = fmaxf(top[e / GROUPS], fmaxf(fabsf(lowest), fabsf(fmaf(15.0f, pair_step(pair[e]), lowest))));
            }
        }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const float all = block_max(top[v], scratch);
        if (threadIdx.x == 0) st_cluster(peer_addr(smem_u32(&every[v][rank]), 0), all);
    }
    const int first = __syncthreads_or(marked & 1), second = __syncthreads_or(marked & 2);
    if (threadIdx.x == 0) st_cluster(peer_addr(smem_u32(&every[2][rank]), 0), (float)((first ? 1 : 0) + (second ? 2 : 0)));
    cluster_sync_all();
    if (rank || threadIdx.x >= 32) return;
    int ahead = 0;                                     // pages of the requests in front of this one
    for (int i = threadIdx.x; i < n; i += 32) ahead += unpack_room(p, i);
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    if (threadIdx.x) return;
    int e[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        float all = 0.0f;
        for (int i = 0; i < PK_CLUSTER; ++i) all = fmaxf(all, every[v][i]);
        e[v] = half_shift(all);
    }
    marked = 0;
    for (int i = 0; i < PK_CLUSTER; ++i) marked |= (int)every[2][i];
    p.written[(size_t)n * p.nkv + kvh] = {e[0], e[1], marked, ahead - lo / PK_WIDE};
}

// The positions that a request's rows read, written out in half precision as the prompt attention takes them, in pages of PK_WIDE whatever the packed ones hold:
// page i of a request where `written` says.  A CTA takes one of those pages of one kv head, a thread a word of 8 codes at a time, all its loads on their way
// together (a CTA for every 16 positions waited for its loads: 16 us for 16,000 positions of 4 kv heads); bound by the bytes written (heads of 128: 144 bytes
// read and 512 written a position and kv head).  Positions behind the request's last are written as noughts: nobody reads them, and no number from nowhere
// stands there.
template <int HD>
__global__ void __launch_bounds__(PK_THREADS) packed_unpack_kernel(const PkUnpack p) {
    constexpr int WORDS = HD / 8, EACH = 2 * PK_WIDE * WORDS / PK_THREADS;
    pdl_launch();
    const int n = blockIdx.z, kvh = blockIdx.y;
    pdl_wait();
    const int req = p.longs[3 * n], row0 = p.longs[3 * n + 1], rows = p.longs[3 * n + 2];
    const int last = p.positions[row0 + rows - 1], lo = first_visible(p.positions[row0], p.window), wide = lo / PK_WIDE + blockIdx.x;
    const PkWritten as = p.written[(size_t)n * p.nkv + kvh];
    const int room = unpack_room(p, n), place = as.base + wide;
    if (blockIdx.x == 0 && kvh == 0 && (last / PK_WIDE - lo / PK_WIDE >= room || last / PK_WIDE >= p.table_pages)) {
        // (positions beyond what the plan or the call's bound says: what there is no room for is not there)
        if (p.status && threadIdx.x == 0) atomicOr(p.status, BG_STATUS_BAD_PAGE);
        for (int i = lo / PK_WIDE + room + threadIdx.x; i < p.table_pages; i += PK_THREADS) p.table[(size_t)n * p.table_pages + i] = -1;
    }
    if (wide > last / PK_WIDE || wide >= p.table_pages || (int)blockIdx.x >= room || place < 0 || place >= p.room) return;
    if (kvh == 0 && threadIdx.x == 0) p.table[(size_t)n * p.table_pages + wide] = place;
    __shared__ const unsigned char* tiles[PK_WIDE / PK_TILE];
    __shared__ unsigned marks[Packed<HD>::GROUPS][PK_WIDE / 32];
    if (threadIdx.x < Packed<HD>::GROUPS * PK_WIDE / 32) marks[threadIdx.x / (PK_WIDE / 32)][threadIdx.x % (PK_WIDE / 32)] = 0;
    if (threadIdx.x < PK_WIDE / PK_TILE) {
        const int pos0 = wide * PK_WIDE + threadIdx.x * PK_TILE, page = unpack_page(p, req, pos0, lo, last, true);
        tiles[threadIdx.x] = page < 0 ? nullptr
            : p.pool + ((size_t)page * p.nkv + kvh) * p.block_bytes + (size_t)(pos0 % p.page_size / PK_TILE) * Packed<HD>::TILE;
    }
    __syncthreads();
    unsigned pair[EACH], word[EACH];
    unsigned have = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {                   // (first the keys of all positions, then their values)
        const int i = j * PK_THREADS + threadIdx.x, value = i / (PK_WIDE * WORDS), slot = i / WORDS % PK_WIDE, f = i % WORDS * 8;
        const unsigned char* from = tiles[slot / PK_TILE];
        pair[j] = word[j] = 0;
        if (!from || wide * PK_WIDE + slot > last) continue;
        pair[j] = *reinterpret_cast<const unsigned*>(from + Packed<HD>::pair_word(slot % PK_TILE, value, f / PK_GROUP));
        word[j] = *reinterpret_cast<const unsigned*>(from + (value ? Packed<HD>::value_word(slot % PK_TILE, f) : Packed<HD>::key_word(slot % PK_TILE, f)));
        have |= 1u << j;
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int i = j * PK_THREADS + threadIdx.x, value = i / (PK_WIDE * WORDS), slot = i / WORDS % PK_WIDE, f = i % WORDS * 8;
        float v[8] = {};
        if (have >> j & 1) {
            if (!value) packed_values<true>(word[j], pair[j], v);
            else if (!as.marked || pair_finite(pair[j])) packed_values<false>(word[j], pair[j], v);
            else atomicOr(&marks[f / PK_GROUP][slot / 32], 1u << (slot % 32));
        }
        const float down = __uint_as_float((unsigned)(127 - (value ? as.values : as.keys)) << 23);
        uint4 r;
        __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(v[2 * e] * down, v[2 * e + 1] * down);
        *reinterpret_cast<uint4*>(p.out + (((size_t)place * 2 + value) * p.nkv + kvh) * PK_WIDE * HD + (size_t)slot * HD + f) = r;
    }
    if (!as.marked) return;
    __syncthreads();
    if (threadIdx.x < Packed<HD>::GROUPS)
        p.marks[((size_t)place * p.nkv + kvh) * Packed<HD>::GROUPS + threadIdx.x] = (unsigned long long)marks[threadIdx.x][1] << 32 | marks[threadIdx.x][0];
}

static int packed_shape(int hd, int page_size, int nkv, int num_pages, long long block_bytes, bool bounds) {
    if (hd != 64 && hd != 128) return BG_ERR_UNSUPPORTED;
    if (page_size <= 0 || page_size % PK_TILE || nkv <= 0 || nkv > 65535 || num_pages <= 0) return BG_ERR_SHAPE;
    if (block_bytes % 16 || block_bytes < page_size / PK_TILE * packed_tile_bytes(hd) + (bounds ? 4 * hd : 0)) return BG_ERR_SHAPE;
    return BG_OK;
}

template <typename TS, typename TQ, int HD>
static int append_launch(const PkAppend& p, cudaStream_t stream) {
    const long long each_q = PK_THREADS / (HD / 16), each = PK_THREADS / (HD / 8);
    const long long queries = ((long long)p.T * p.nh + each_q - 1) / each_q, others = ((long long)p.T * 2 * p.nkv + each - 1) / each;
    if (queries + others > 0x7fffffffLL) return BG_ERR_SHAPE;
    const dim3 grid((unsigned)(queries + others));
    // (halves of whole pieces of 8 features, whose table rows are whole float4s)
    const bool split = !p.interleaved && p.rot % 16 == 0 && (uintptr_t)p.cos_sin % 16 == 0;
    cudaError_t e = split ? launch(packed_append_kernel<TS, TQ, HD, true>, grid, dim3(PK_THREADS), 0, stream, p, (int)others)
                          : launch(packed_append_kernel<TS, TQ, HD, false>, grid, dim3(PK_THREADS), 0, stream, p, (int)others);
    return e == cudaSuccess ? BG_OK : (int)e;
}

}  // namespace bg

using namespace bg;

// Bytes of a tile of 16 positions of one kv head, or a negative code.
extern "C" int bg_packed_tile_bytes(int hd) { return hd == 64 || hd == 128 ? (int)packed_tile_bytes(hd) : BG_ERR_UNSUPPORTED; }

// Bytes of the calls' fields: 0 an append, 1 a reading call.
extern "C" int bg_packed_call_bytes(int which) { return which == 0 ? (int)sizeof(PkAppend) : (int)sizeof(PkRead); }

extern "C" int bg_packed_append(const void* call, cudaStream_t stream) {
    const PkAppend& p = *(const PkAppend*)call;
    if (int e = packed_shape(p.hd, p.page_size, p.nkv, p.num_pages, p.block_bytes, false)) return e;
    if (p.T <= 0) return BG_OK;
    if (p.parts < 1 || p.nh <= 0 || p.rot < 0 || p.rot > p.hd || p.rot % 2 || p.max_pages <= 0 || (p.rot && !p.cos_sin)) return BG_ERR_SHAPE;
    const long long size = p.src_dtype == BG_DTYPE_F32 ? 4 : 2, size_q = p.q_dtype == BG_DTYPE_F32 ? 4 : 2;
    if (((long long)(uintptr_t)p.src | p.src_stride * size | (p.parts > 1 ? p.part_stride * size : 0)) & 15
        || ((long long)(uintptr_t)p.q_out | p.q_stride * size_q) & 15 || (uintptr_t)p.pool % 16 || (uintptr_t)p.cos_sin % 8) return BG_ERR_ALIGN;
    BG_DISPATCH_DTYPE(p.src_dtype, TS, BG_DISPATCH_DTYPE(p.q_dtype, TQ, return p.hd == 64 ? (append_launch<TS, TQ, 64>(p, stream)) : (append_launch<TS, TQ, 128>(p, stream))));
}

extern "C" int bg_packed_rows(const void* call, cudaStream_t stream) {
    const PkRead& p = *(const PkRead*)call;
    if (int e = packed_shape(p.hd, p.page_size, p.nkv, p.num_pages, p.block_bytes, false)) return e;
    if (p.T <= 0) return BG_OK;
    if ((uintptr_t)p.pool % 16 || (uintptr_t)p.out % 16) return BG_ERR_ALIGN;
    const dim3 grid(p.T, (2 * p.nkv * p.hd / 8 + PK_THREADS - 1) / PK_THREADS);
    cudaError_t e = cudaSuccess;
    BG_DISPATCH_DTYPE(p.out_dtype, TO, e = p.hd == 64 ? launch(packed_rows_kernel<TO, 64>, grid, dim3(PK_THREADS), 0, stream, p)
                                                      : launch(packed_rows_kernel<TO, 128>, grid, dim3(PK_THREADS), 0, stream, p));
    return e == cudaSuccess ? BG_OK : (int)e;
}

extern "C" int bg_packed_bounds(const void* call, cudaStream_t stream) {
    const PkRead& p = *(const PkRead*)call;
    if (int e = packed_shape(p.hd, p.page_size, p.nkv, p.num_pages, p.block_bytes, true)) return e;
    if (p.T <= 0) return BG_OK;
    if ((uintptr_t)p.pool % 16) return BG_ERR_ALIGN;
    const dim3 grid((p.T + PK_ROWS - 1) / PK_ROWS, p.nkv);
    cudaError_t e = p.hd == 64 ? launch(packed_bounds_kernel<64>, grid, dim3(PK_THREADS), 0, stream, p)
                               : launch(packed_bounds_kernel<128>, grid, dim3(PK_THREADS), 0, stream, p);
    return e == cudaSuccess ? BG_OK : (int)e;
}

// Positions of a page that bg_packed_unpack writes.
extern "C" int bg_packed_wide_page() { return PK_WIDE; }

// Pages of them that `rows` rows need whose positions lie below `end`.
extern "C" int bg_packed_room(int rows, int end, int window) { return packed_room(rows, end, window); }

// Pages in half precision for the prompt attention.  out [room, ..] holds the requests' pages one behind the other, bg_packed_room() of each (most_pages the most
// of one); table [n][table_pages] their numbers.  `ends` or `end` bound the positions; a request that goes on beyond them has the status say so.

extern "C" int bg_packed_unpack(const unsigned char* pool, long long block_bytes, int num_pages, int page_size, const int* positions, const int* block_table,
                                int max_pages, int n_req, const int* longs, const int* ends, int n, void* out, int* table, void* written, void* marks,
                                int most_pages, int table_pages, int room, int end, int window, int nkv, int hd, unsigned* status, cudaStream_t stream) {
    if (int e = packed_shape(hd, page_size, nkv, num_pages, block_bytes, false)) return e;
    if (n <= 0) return BG_OK;
    if (n > 65535 || most_pages <= 0 || table_pages < most_pages || room < most_pages || table_pages > 0x7fffffff / PK_WIDE || end <= 0) return BG_ERR_SHAPE;
    if ((uintptr_t)pool % 16 || (uintptr_t)out % 16 || (uintptr_t)written % 16 || (uintptr_t)marks % 8) return BG_ERR_ALIGN;
    const PkUnpack p = {pool, block_bytes, positions, block_table, longs, ends, (__half*)out, table, (PkWritten*)written, (unsigned long long*)marks, max_pages,
                        num_pages, page_size, n_req, nkv, table_pages, room, end, window, status};
    const dim3 heads(nkv, n, PK_CLUSTER), whole(most_pages, nkv, n);
    cudaError_t e = hd == 64 ? launch_cluster(packed_reach_kernel<64>, heads, dim3(PK_THREADS), 0, stream, PK_CLUSTER, p)
                             : launch_cluster(packed_reach_kernel<128>, heads, dim3(PK_THREADS), 0, stream, PK_CLUSTER, p);
    if (e != cudaSuccess) return (int)e;
    e = hd == 64 ? launch(packed_unpack_kernel<64>, whole, dim3(PK_THREADS), 0, stream, p) : launch(packed_unpack_kernel<128>, whole, dim3(PK_THREADS), 0, stream, p);
    return e == cudaSuccess ? BG_OK : (int)e;
}
