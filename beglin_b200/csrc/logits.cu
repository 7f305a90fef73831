// What is done to a row of logits before a token is chosen from it: penalties for tokens that the request holds already,
// biases of single tokens, and a mask of the tokens that are allowed.
//
// For a token v that occurs in the request's text, c times of them in the part that was generated:
//   x > 0: x / repetition, else x * repetition;     x -= frequency c;     x -= presence  where c > 0
// then x += bias[v], and a token that the mask does not allow becomes -inf.
//
// A CTA takes a range of one row's vocabulary.  It counts the tokens of the text that lie in its range in shared memory (a word a
// token: bit 31 for one of the prompt, the others count the generated ones), so the text is read once a range from the L2 and
// the row once from memory; the order of the counts does not matter, so results do not depend on it.  A group of four tokens that the
// mask excludes is not read, and in place a group that nothing changes is not written.
#include "common.cuh"

namespace bg {

struct LogitsParams {
    const float* x;
    long long ldx;
    float* out;
    long long ldo;
    int V;
    int* history;               // [n][cap] the tokens that a request holds, in order, or null
    int cap;
    const int* lengths;         // [n] how many, without `newest`
    const int* prompts;         // [n] how many of them are the prompt's, or null: all are generated
    const int* newest;          // [n] one more token, stored at history[r][lengths[r]] for the steps to come, or null
    const float *repetition, *frequency, *presence;      // [n], or null: 1, 0, 0
    const int* bias_id;         // the rows' biased tokens, ascending in each row, or null
    const float* bias;
    const int* bias_row;        // [n + 1] where a row's begin
    const unsigned* allowed;    // [masks][words], bit v % 32 of word v / 32, or null
    int words;
    const int* allowed_row;     // [n] a row's mask, -1: none; or null: mask r for row r
    int masks;
    unsigned* status;
};

// VEC: tokens of a load (4 where rows begin on 16 bytes).  A CTA's range: THREADS x LOADS x VEC tokens.
template <int THREADS, int LOADS, int VEC>
__global__ void __launch_bounds__(THREADS) adjust_logits_kernel(LogitsParams p) {
    constexpr int RANGE = THREADS * LOADS * VEC;
    extern __shared__ unsigned count_s[];              // [RANGE]
    pdl_launch();
    pdl_wait();
    const int r = blockIdx.y, tid = threadIdx.x;
    const int v0 = blockIdx.x * RANGE, v1 = min(p.V, v0 + RANGE);
    const float* x = p.x + (size_t)r * p.ldx;
    float* out = p.out + (size_t)r * p.ldo;
    const bool in_place = x == out;
    const float rep = p.repetition ? p.repetition[r] : 1.0f, freq = p.frequency ? p.frequency[r] : 0.0f, pres = p.presence ? p.presence[r] : 0.0f;
    int len = p.history ? min(max(p.lengths[r], 0), p.cap) : 0;
    const int prompt = p.prompts ? p.prompts[r] : 0;
    const int newest = p.newest ? p.newest[r] : -1;
    const int mask_row = p.allowed ? (p.allowed_row ? p.allowed_row[r] : r) : -1;
    const bool masked = mask_row >= 0 && mask_row < p.masks;
    if (mask_row >= p.masks && p.allowed && tid == 0 && p.status) atomicOr(p.status, BG_STATUS_BAD_TOKEN);
    const unsigned* mask = p.allowed + (masked ? (size_t)mask_row * p.words : 0);
    const bool counts = (rep != 1.0f || freq != 0.0f || pres != 0.0f) && (len > 0 || newest >= 0);

    // ---- the row's values on their way, behind the mask where there is one
    float v[LOADS][VEC];
    unsigned ok[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = v0 + (i * THREADS + tid) * VEC;
        ok[i] = at < v1 ? (masked ? mask[at >> 5] >> (at & 31) : 0xffffffffu) : 0u;
        ok[i] &= (1u << VEC) - 1;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = v0 + (i * THREADS + tid) * VEC;
        if constexpr (VEC == 4) {
            float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (ok[i]) {
                if (at + 4 <= v1) f = *reinterpret_cast<const float4*>(x + at);
                else { f.x = x[at]; if (at + 1 < v1) f.y = x[at + 1]; if (at + 2 < v1) f.z = x[at + 2]; }
            }
            v[i][0] = f.x; v[i][1] = f.y; v[i][2] = f.z; v[i][3] = f.w;
        } else {
            v[i][0] = ok[i] ? x[at] : -INFINITY;
        }
    }

    // ---- the tokens that the request holds
    int* history = p.history ? p.history + (size_t)r * p.cap : nullptr;
    if (history && p.newest && blockIdx.x == 0 && tid == 0) {
        if (newest >= 0 && newest < p.V && len < p.cap) history[len] = newest;         // (no CTA of the row reads this place)
        else if (p.status) atomicOr(p.status, BG_STATUS_BAD_TOKEN);
    }
    if (counts) {
        for (int i = tid * 4; i < RANGE; i += THREADS * 4) *reinterpret_cast<uint4*>(count_s + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto hold = [&](int id, bool given) {
            if ((unsigned)id >= (unsigned)p.V) { if (p.status) atomicOr(p.status, BG_STATUS_BAD_TOKEN); return; }
            if (id < v0 || id >= v1) return;
            if (given) atomicOr(&count_s[id - v0], 0x80000000u); else atomicAdd(&count_s[id - v0], 1u);
        };
        for (int i = tid; i < len; i += THREADS) hold(history[i], i < prompt);
        if (tid == 0 && p.newest) hold(newest, false);
        __syncthreads();
    }

#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int local = (i * THREADS + tid) * VEC, at = v0 + local;
        if (at >= v1) continue;
        bool changed = !in_place;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const unsigned c = counts ? count_s[local + j] : 0u;
            const bool allowed = ok[i] >> j & 1;
            if (c) {
                float y = v[i][j];
                y = y > 0.0f ? y / rep : y * rep;
                const unsigned made = c & 0x7fffffffu;
                if (made) { y -= freq * (float)made; y -= pres; }
                v[i][j] = y;
                changed = true;
            }
            if (!allowed) { v[i][j] = -INFINITY; changed = true; }
        }
        if (!changed) continue;
        if constexpr (VEC == 4) {
            if (at + 4 <= v1) *reinterpret_cast<float4*>(out + at) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
            else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < v1) out[at + j] = v[i][j];
            }
        } else {
            out[at] = v[i][0];
        }
    }

    // ---- the few biased tokens, on what has just been written
    if (p.bias_id) {
        __syncthreads();
        const int b0 = p.bias_row[r], b1 = p.bias_row[r + 1];
        for (int i = b0 + tid; i < b1; i += THREADS) {
            const int id = p.bias_id[i], before = i > b0 ? p.bias_id[i - 1] : -1;
            if ((unsigned)id >= (unsigned)p.V || before > id) { if (p.status) atomicOr(p.status, BG_STATUS_BAD_TOKEN); continue; }
            if (id < v0 || id >= v1 || id == before) continue;                          // (a token's first entry adds all of its entries)
            if (masked && !(mask[id >> 5] >> (id & 31) & 1)) continue;
            float y = out[id];
            for (int j = i; j < b1 && p.bias_id[j] == id; ++j) y += p.bias[j];
            out[id] = y;
        }
    }
}

template <int THREADS, int LOADS, int VEC>
static int al_launch(const LogitsParams& p, int n, cudaStream_t stream) {
    constexpr int range = THREADS * LOADS * VEC;
    auto kern = adjust_logits_kernel<THREADS, LOADS, VEC>;
    if (range * 4 >= BG_SMEM_OPT_IN) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, range * 4);
        if (e != cudaSuccess) return (int)e;
    }
    cudaError_t e = launch(kern, dim3((unsigned)((p.V + range - 1) / range), (unsigned)n), dim3(THREADS), (size_t)range * 4, stream, p);
    return e == cudaSuccess ? BG_OK : (int)e;
}

}  // namespace bg

using namespace bg;

// See the head of this file; `out` may be `x`.  A token outside [0, V), a row's biased tokens out of order and a mask that is not there
// set BG_STATUS_BAD_TOKEN and are passed over.
extern "C" int bg_adjust_logits(const float* x, long long ldx, float* out, long long ldo, int n, int V, int* history, int cap, const int* lengths,
                                const int* prompts, const int* newest, const float* repetition, const float* frequency, const float* presence,
                                const int* bias_id, const float* bias, const int* bias_row, const int* allowed, int words, const int* allowed_row,
                                int masks, unsigned* status, cudaStream_t stream) {
    if (n <= 0) return BG_OK;
    if (V <= 0 || n > 65535 || ldx < V || ldo < V || (history && (!lengths || cap <= 0)) || (newest && !history)) return BG_ERR_SHAPE;
    if ((bias_id && (!bias || !bias_row)) || (allowed && (words < (V + 31) / 32 || masks <= 0))) return BG_ERR_SHAPE;
    if (V > 0x7fffffff - 65536) return BG_ERR_SHAPE;
    LogitsParams p{x, ldx, out, ldo, V, history, cap, lengths, prompts, newest, repetition, frequency, presence, bias_id, bias, bias_row,
                   (const unsigned*)allowed, words, allowed_row, masks, status};
    const bool pieces = ldx % 4 == 0 && ldo % 4 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)out % 16 == 0;
    if (pieces) return al_launch<256, 4, 4>(p, n, stream);
    return al_launch<256, 16, 1>(p, n, stream);
}
