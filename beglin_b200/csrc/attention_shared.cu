// Attention of single tokens whose requests share their first positions, in three parts: the shared positions, read once for all rows of a group
// (attention_tcgen05.cu, SHARED), each request's own positions behind them (attention_mma.cu, SHARED), and here the joining of a row's partial results:
//   m = max_i m_i,   out = sum_i o_i e^(m_i - m) / sum_i l_i e^(m_i - m),
// over the slots 0 .. n - 1 of the row's group and those of the ranges that its own positions are cut into.
#include "common.cuh"

// How a layer's attention goes over shared positions, and what a step brings to it.  The host side fills the fields by name.
struct SharedAttnArgs {
    const int* items;           // [n_items][8], as the kernel of the shared positions takes them
    const int* rows;
    const int* own_first;       // [T] tensor cores: a row's first position of its own
    const int* parts;           // [T] tensor cores: results of a row over what it shares
    int tensor_cores, T, nh, nkv, hd, vd, page_size, q_dtype, cache_dtype, n_items;
    int slots;                  // the most results of a row over what it shares
    int split, tile, bq;        // float units: keys of a split and a tile, rows of a block
};
struct SharedAttnStep {
    const void* q; const void* pool; const int* table; const int* positions; void* out; const float* sink_w; unsigned* status; float* scratch;
    long long scratch_floats;
    int q_stride, out_stride, max_pages, num_pages;
    int ranges;                 // tensor cores: ranges that a row's own positions are cut into; float units: splits of the longest row
    int at_once;                // float units: the most splits of a block
    int sink, out_dtype;
    float scale, softcap;
};

namespace bg {

// WARPS warps take one (row, head), a lane four neighbouring features; warp w joins the slots w, w + WARPS, ...
// eight at a time, all on their way together, and the warps' results are joined in their order.  Which slots a warp takes hangs on the slots' numbers alone.
constexpr int SM_THREADS = 256;
template <int HD, int WARPS>
__global__ void __launch_bounds__(SM_THREADS)
attention_shared_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ positions,
                              const int* __restrict__ own_first, const int* __restrict__ shared_slots, int T, int nh, int slots, int first_slot,
                              int n_own, const float* __restrict__ sink_w, int sink, __nv_bfloat16* __restrict__ out, int out_stride) {
    constexpr int AT_ONCE = 8, GROUPS = SM_THREADS / 32 / WARPS;       // (row, head) pairs of a CTA
    __shared__ float4 acc_s[WARPS > 1 ? SM_THREADS / 32 : 1][32];
    __shared__ float2 ml_s[WARPS > 1 ? SM_THREADS / 32 : 1];
    pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WARPS;
    const int w = blockIdx.x * GROUPS + warp / WARPS;
    const bool idle = w >= T * nh;
    const int t = idle ? 0 : w / nh, h = w - t * nh;
    const int n_shared = shared_slots[t];
    const int own = positions[t] + 1 - own_first[t];
    const int range = keys_per_split(0, own, n_own);
    const int n = idle ? 0 : n_shared + (own > 0 ? (own + range - 1) / range : 0);
    pdl_wait();
    const size_t base = (size_t)w * slots;
    const int d = lane * 4;
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = part; i0 < n; i0 += AT_ONCE * WARPS) {
        float2 ml[AT_ONCE];
        float4 v[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int i = i0 + j * WARPS;
            const bool have = i < n;
            const size_t slot = base + (i < n_shared ? i : first_slot + i - n_shared);
            ml[j] = have ? *reinterpret_cast<const float2*>(part_ml + slot * 2) : make_float2(-INFINITY, 0.0f);
            v[j] = have && d < HD ? *reinterpret_cast<const float4*>(part_o + slot * HD + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) top = fmaxf(top, ml[j].x);
        if (top == -INFINITY) {                        // no position seen so far, or scores that are no numbers: those have no maximum, and show by their sum
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) l += ml[j].y;
            continue;
        }
        const float keep = expf(m - top);
        l *= keep; acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
        m = top;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const float f = ml[j].x == -INFINITY ? 0.0f : expf(ml[j].x - m);
            l = fmaf(ml[j].y, f, l);
            acc.x = fmaf(v[j].x, f, acc.x); acc.y = fmaf(v[j].y, f, acc.y); acc.z = fmaf(v[j].z, f, acc.z); acc.w = fmaf(v[j].w, f, acc.w);
        }
    }
    if constexpr (WARPS > 1) {
        acc_s[warp][lane] = acc;
        if (lane == 0) ml_s[warp] = make_float2(m, l);
        __syncthreads();
        if (part) return;
    }
    if (idle || d >= HD) return;
    const float sv = sink && sink_w ? sink_w[h] : 0.0f;
    float top = sink ? fmaxf(m, sv) : m;
    if constexpr (WARPS > 1) {
#pragma unroll
        for (int j = 1; j < WARPS; ++j) top = fmaxf(top, ml_s[warp + j].x);
    }
    const float f0 = m == -INFINITY ? 0.0f : expf(m - top);
    float sum = fmaf(l, f0, sink ? expf(sv - top) : 0.0f);
    float4 o = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
    if constexpr (WARPS > 1) {
#pragma unroll
        for (int j = 1; j < WARPS; ++j) {
            const float2 ml = ml_s[warp + j];
            const float4 v = acc_s[warp + j][lane];
            const float f = ml.x == -INFINITY ? 0.0f : expf(ml.x - top);
            sum = fmaf(ml.y, f, sum);
            o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;          // (a row that sees nothing is nought)
    const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * inv, o.y * inv), y = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(out + (size_t)t * out_stride + (size_t)h * HD + d) =
        make_uint2(*reinterpret_cast<const unsigned*>(&x), *reinterpret_cast<const unsigned*>(&y));
}

}  // namespace bg

using namespace bg;

// Joins the partial results of bg_attention_tc_shared (slots 0 .. parts[t] - 1 of row t) and bg_attention_mma_own (n_own ranges from first_slot on).
static int shared_merge(const float* part_o, const float* part_ml, const int* positions, const int* own_first, const int* parts, int T, int nh, int hd, int slots,
                        int first_slot, int n_own, int sink, const float* sink_w, void* out, int out_stride, cudaStream_t stream) {
    if (first_slot + n_own > slots || (long long)T * nh > 0x7fffffff - 64) return BG_ERR_SHAPE;
    if (out_stride % 4 || (uintptr_t)out % 8) return BG_ERR_ALIGN;
    // more warps to a (row, head) where slots are many and rows few
    const int warps = slots > 8 ? 4 : 1, groups = SM_THREADS / 32 / warps;
    auto kern = hd == 128 ? (warps > 1 ? attention_shared_merge_kernel<128, 4> : attention_shared_merge_kernel<128, 1>)
                          : (warps > 1 ? attention_shared_merge_kernel<64, 4> : attention_shared_merge_kernel<64, 1>);
    cudaError_t e = launch(kern, dim3((unsigned)(((long long)T * nh + groups - 1) / groups)), dim3(SM_THREADS), 0, stream, part_o, part_ml, positions, own_first,
                           parts, T, nh, slots, first_slot, n_own, sink_w, sink, (__nv_bfloat16*)out, out_stride);
    return e == cudaSuccess ? BG_OK : (int)e;
}

// Bytes of what the host side mirrors field by field; it compares them when it loads the library.
extern "C" int bg_shared_attention_bytes(int step) { return (int)(step ? sizeof(SharedAttnStep) : sizeof(SharedAttnArgs)); }

// The whole attention of a step of single tokens over shared and own positions, as one call.  scratch: T * nh * n * (vd + 2) floats, n the float units' `ranges`
// or the tensor cores' slots + ranges (none where nothing is shared and there is one range).
extern "C" int bg_shared_attention(const SharedAttnArgs* args, const SharedAttnStep* step, cudaStream_t stream) {
    const SharedAttnArgs& a = *args;
    const SharedAttnStep& s = *step;
    if (a.T <= 0) return BG_OK;
    if (a.nh <= 0 || a.nkv <= 0 || a.nh % a.nkv || a.hd <= 0 || a.vd <= 0 || s.ranges <= 0 || a.slots < 0 || (uintptr_t)s.scratch % 16) return BG_ERR_SHAPE;
    const long long results = a.tensor_cores && !a.n_items && s.ranges == 1 ? 0 : (long long)a.T * a.nh * (a.tensor_cores ? a.slots + s.ranges : s.ranges);
    if (s.scratch_floats < results * (a.vd + 2)) return BG_ERR_SHAPE;
    float *part_o = s.scratch, *part_ml = s.scratch + results * a.vd;
    if (!a.tensor_cores) {
        int rc = bg_attention_shared_partial(s.q, a.q_dtype, s.q_stride, s.pool, a.cache_dtype, s.num_pages, a.page_size, s.table, s.max_pages, s.positions, a.items,
                                             a.n_items, a.rows, part_o, part_ml, s.ranges, s.at_once, a.nh, a.nkv, a.hd, a.vd, a.split, a.tile, a.bq, s.scale,
                                             s.softcap, s.status, stream);
        if (rc != BG_OK) return rc;
        return bg_attention_merge(part_o, part_ml, s.positions, s.out, s.out_dtype, s.out_stride, a.T, a.nh, a.vd, s.ranges, a.split, 0, s.sink, s.sink_w, 0, stream);
    }
    if (a.q_dtype != BG_DTYPE_BF16 || a.cache_dtype != BG_DTYPE_BF16 || s.out_dtype != BG_DTYPE_BF16) return BG_ERR_DTYPE;
    if (!a.n_items && s.ranges == 1)                 // nothing is shared, and a CTA walks all of a row's positions: one kernel, which writes the rows
        return bg_attention_mma_own(s.q, s.q_stride, s.pool, s.num_pages, a.page_size, s.table, s.max_pages, s.positions, a.own_first, a.T, nullptr, nullptr, 1, 0, 1,
                                    a.nh, a.nkv, a.hd, s.scale, s.softcap, 0, s.out, s.out_stride, s.sink, s.sink_w, s.status, stream);
    const int slots = a.slots + s.ranges;
    int rc = bg_attention_tc_shared(s.q, s.q_stride, s.pool, s.num_pages, a.page_size, s.table, s.max_pages, s.positions, a.items, a.n_items, a.rows, part_o,
                                    part_ml, slots, a.nh, a.nkv, a.hd, s.scale, s.softcap, s.status, stream);
    if (rc == BG_OK)
        rc = bg_attention_mma_own(s.q, s.q_stride, s.pool, s.num_pages, a.page_size, s.table, s.max_pages, s.positions, a.own_first, a.T, part_o, part_ml, slots,
                                  a.slots, s.ranges, a.nh, a.nkv, a.hd, s.scale, s.softcap, a.n_items > 0, nullptr, 0, 0, nullptr, s.status, stream);
    if (rc == BG_OK)
        rc = shared_merge(part_o, part_ml, s.positions, a.own_first, a.parts, a.T, a.nh, a.hd, slots, a.slots, s.ranges, s.sink, s.sink_w, s.out, s.out_stride,
                          stream);
    return rc;
}
