// What is done to a row of logits before a token is chosen from it: penalties for tokens that the request holds already,
// biases of single tokens, and a mask of the tokens that are allowed.
//
// For a token v that occurs in the request's text, c times of them in the part that was generated:
//   x > 0: x / repetition, else x * repetition;     x -= frequency c;     x -= presence  where c > 0
// then x += bias[v], and a token that the mask does not allow becomes -inf.
//
// Two kinds of work.  A row's copy, with -inf where the mask says so (a group of four tokens that the mask excludes is not read; in place only what the mask
// excludes is written): bound by memory.  And the mending of the tokens that the text or the biases name: a CTA takes a range of one row's vocabulary, counts
// those that lie in it in shared memory (a word a token: bit 31 for one of the prompt, bit 30 for a biased one, the others count the generated ones), and
// whoever takes a token's word first mends the token, so the order of the counts does not matter.  Every CTA reads the whole text (from the L2), which is
// what mending costs: few rows do both in one kernel, with ranges small enough for all SMs; many rows copy first and mend then, a text's words in a table of
// its tokens in place of a range of the vocabulary.  64 rows of 151,936 with 2,048 to 4,096 tokens of text, 300 biases and masks for half of them: 22 us, 13.3
// of them the copy (a plain copy takes 13.6); 25 with words for ranges of 16,384 tokens, 51 in one kernel.  One row with 700: 2.6 us in one kernel, 5.9 in
// two.  What bounds the mending is a chain: lengths, text, counts, values (4.8 us for texts of 100, some 2,000 cycles more for every 1,024).
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
    const int* prompts;         // [n] how many of them, `newest` among them, are the prompt's, or null: all are generated
    const int* newest;          // [n] one more token, stored at history[r][lengths[r]] for the steps to come, or null
    const float *repetition, *frequency, *presence;      // [n], or null: 1, 0, 0
    const int* bias_id;         // the rows' biased tokens, ascending in each row, or null
    const float* bias;
    const int* bias_row;        // [n + 1] where a row's begin
    int n_bias;                 // how many there are in all
    const unsigned* allowed;    // [masks][words], bit v % 32 of word v / 32, or null
    int words;
    const int* allowed_row;     // [n] a row's mask, -1: none; or null: mask r for row r
    int masks;
    unsigned* status;
};

// What a CTA knows of its row.
struct LogitsRow {
    const float* x;
    float* out;
    const unsigned* mask;       // null: every token is allowed
    int* history;
    float rep, freq, pres;
    int len, prompt, newest, b0, b1;
    bool counts;                // penalties: the text counts
    __device__ __forceinline__ LogitsRow(const LogitsParams& p, int r) {
        x = p.x + (size_t)r * p.ldx;
        out = p.out + (size_t)r * p.ldo;
        rep = p.repetition ? p.repetition[r] : 1.0f; freq = p.frequency ? p.frequency[r] : 0.0f; pres = p.presence ? p.presence[r] : 0.0f;
        len = p.history ? min(max(p.lengths[r], 0), p.cap) : 0;
        prompt = p.prompts ? p.prompts[r] : 0;
        newest = p.newest ? p.newest[r] : -1;
        history = p.history ? p.history + (size_t)r * p.cap : nullptr;
        b0 = p.bias_id ? min(max(p.bias_row[r], 0), p.n_bias) : 0;
        b1 = p.bias_id ? min(max(p.bias_row[r + 1], 0), p.n_bias) : 0;
        const int m = p.allowed ? (p.allowed_row ? p.allowed_row[r] : r) : -1;
        mask = m >= 0 && m < p.masks ? p.allowed + (size_t)m * p.words : nullptr;
        if (m >= p.masks && p.allowed && threadIdx.x == 0 && p.status) atomicOr(p.status, BG_STATUS_BAD_TOKEN);
        counts = (rep != 1.0f || freq != 0.0f || pres != 0.0f) && (len > 0 || newest >= 0);
    }
    __device__ __forceinline__ bool allows(int id) const { return !mask || (mask[id >> 5] >> (id & 31) & 1); }
};

// The tokens v0 .. v1 - 1 of a row on their way into registers, and from there to `out`.  VEC: tokens of a load (4 where rows begin on 16 bytes).
template <int THREADS, int LOADS, int VEC>
struct LogitsRange {
    static constexpr int RANGE = THREADS * LOADS * VEC;
    static constexpr unsigned ALL = (1u << VEC) - 1;
    float v[LOADS][VEC];
    unsigned ok[LOADS];
    __device__ __forceinline__ void load(const LogitsRow& w, int v0, int v1) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = v0 + (i * THREADS + (int)threadIdx.x) * VEC;
            ok[i] = at < v1 ? (w.mask ? w.mask[at >> 5] >> (at & 31) : ALL) & ALL : 0u;
        }
        if (w.x == w.out) return;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = v0 + (i * THREADS + (int)threadIdx.x) * VEC;
            if constexpr (VEC == 4) {
                float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (ok[i]) {
                    if (at + 4 <= v1) f = *reinterpret_cast<const float4*>(w.x + at);
                    else { f.x = w.x[at]; if (at + 1 < v1) f.y = w.x[at + 1]; if (at + 2 < v1) f.z = w.x[at + 2]; }
                }
                v[i][0] = f.x; v[i][1] = f.y; v[i][2] = f.z; v[i][3] = f.w;
            } else {
                v[i][0] = ok[i] ? w.x[at] : -INFINITY;
            }
        }
    }
    __device__ __forceinline__ void store(const LogitsRow& w, int v0, int v1) {
        const bool in_place = w.x == w.out;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = v0 + (i * THREADS + (int)threadIdx.x) * VEC;
            if (at >= v1 || (in_place && ok[i] == ALL)) continue;
            if (in_place) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (!(ok[i] >> j & 1) && at + j < v1) w.out[at + j] = -INFINITY;
                continue;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (!(ok[i] >> j & 1)) v[i][j] = -INFINITY;
            if constexpr (VEC == 4) {
                if (at + 4 <= v1) *reinterpret_cast<float4*>(w.out + at) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
                else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (at + j < v1) w.out[at + j] = v[i][j];
                }
            } else {
                w.out[at] = v[i][0];
            }
        }
    }
};

// The words of the tokens v0 .. v1 - 1, a token's own at its place ...
struct LogitsDense {
    unsigned* word_s;
    int v0, v1;
    template <int THREADS> __device__ __forceinline__ void clear(int range) {
        for (int i = (int)threadIdx.x * 4; i < range; i += THREADS * 4) *reinterpret_cast<uint4*>(word_s + i) = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ bool owns(int id) const { return id >= v0 && id < v1; }
    __device__ __forceinline__ unsigned* add(int id) { return word_s + (id - v0); }
    __device__ __forceinline__ unsigned* find(int id) { return add(id); }
};
// ... or of a text's tokens wherever they lie in the vocabulary: a table of 2^bits tokens and words with open addresses, larger than the text by a third at
// least, so that a search ends.  Several CTAs share a row's tokens by their low bits.
struct LogitsTable {
    int* key_s;
    unsigned* word_s;
    int bits, part, parts;     // parts: a power of two
    __device__ __forceinline__ bool owns(int id) const { return (id & (parts - 1)) == part; }
    template <int THREADS> __device__ __forceinline__ void clear(int) {
        for (int i = (int)threadIdx.x * 4; i < (1 << bits); i += THREADS * 4) {
            *reinterpret_cast<int4*>(key_s + i) = make_int4(-1, -1, -1, -1);
            *reinterpret_cast<uint4*>(word_s + i) = make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ unsigned first(int id) const { return ((unsigned)id * 2654435761u) >> (32 - bits); }      // (2^32 over the golden ratio)
    __device__ __forceinline__ unsigned* add(int id) {
        for (unsigned h = first(id);; h = (h + 1) & ((1u << bits) - 1)) {
            const int k = atomicCAS(&key_s[h], -1, id);
            if (k == -1 || k == id) return word_s + h;
        }
    }
    __device__ __forceinline__ unsigned* find(int id) {
        for (unsigned h = first(id);; h = (h + 1) & ((1u << bits) - 1)) {
            const int k = key_s[h];
            if (k == id) return word_s + h;
            if (k == -1) return nullptr;
        }
    }
};

// The mending of the tokens that have words.  A biased token without a word (TABLE: it does not occur in the text) is mended by itself.
template <int THREADS, typename WORDS>
struct LogitsMend {
    static constexpr int AHEAD = 8;                    // tokens of the text that a thread has on their way
    static constexpr bool TABLE = !(sizeof(WORDS) == sizeof(LogitsDense) && __is_same(WORDS, LogitsDense));
    const LogitsParams& p;
    const LogitsRow& w;
    WORDS words;
    const int tid, b_at;
    int held[AHEAD], b_id, b_before;
    __device__ __forceinline__ LogitsMend(const LogitsParams& p_, const LogitsRow& w_, const WORDS& words_)
        : p(p_), w(w_), words(words_), tid((int)threadIdx.x), b_at(w_.b0 + (int)threadIdx.x) {}
    __device__ __forceinline__ void bad() const { if (p.status) atomicOr(p.status, BG_STATUS_BAD_TOKEN); }
    __device__ __forceinline__ bool real(int id) const { return (unsigned)id < (unsigned)p.V; }
    __device__ __forceinline__ void fetch_text(int first) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = first + j * THREADS + tid;
            held[j] = i < w.len ? w.history[i] : -1;
        }
    }
    // the first tokens of the text and of the biases on their way
    __device__ __forceinline__ void fetch() {
        if (w.counts) fetch_text(0);
        b_id = b_at < w.b1 ? p.bias_id[b_at] : -1;
        b_before = b_at < w.b1 && b_at > w.b0 ? p.bias_id[b_at - 1] : -1;
    }
    // (with a barrier in front, behind the words' clearing)
    __device__ __forceinline__ void count() {
        auto hold = [&](int id, bool given) {
            if (!real(id)) { bad(); return; }
            if (!words.owns(id)) return;
            unsigned* word = words.add(id);
            if (given) atomicOr(word, 0x80000000u); else atomicAdd(word, 1u);
        };
        if (w.counts) {
            for (int first = 0; first < w.len; first += AHEAD * THREADS) {
                if (first) fetch_text(first);
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const int i = first + j * THREADS + tid;
                    if (i < w.len) hold(held[j], i < w.prompt);
                }
            }
            if (tid == 0 && p.newest) hold(w.newest, w.len < w.prompt);
        }
        for (int i = b_at; i < w.b1; i += THREADS) {
            const int id = i == b_at ? b_id : p.bias_id[i], before = i == b_at ? b_before : p.bias_id[i - 1];
            if (!real(id) || before > id) { bad(); continue; }
            if constexpr (!TABLE) { if (words.owns(id)) atomicOr(words.add(id), 0x40000000u); }
        }
    }
    // Whether a token has a value of its own, and which.  word: what is counted of it; entry: a place among the biased tokens at or before its first, or -1.
    __device__ __forceinline__ bool value(int id, unsigned word, int entry, float& y) const {
        if (!word || !w.allows(id)) return false;
        y = w.x[id];
        const unsigned made = word & 0x3fffffffu;
        if (word & 0xbfffffffu) y = y > 0.0f ? y / w.rep : y * w.rep;
        if (made) { y -= w.freq * (float)made; y -= w.pres; }
        if (word & 0x40000000u) {
            int lo = entry;
            if (lo < 0) {
                lo = w.b0;
                for (int hi = w.b1; lo < hi;) { const int mid = (lo + hi) >> 1; if (p.bias_id[mid] < id) lo = mid + 1; else hi = mid; }
            }
            for (; lo < w.b1 && p.bias_id[lo] == id; ++lo) y += p.bias[lo];     // (its entries lie side by side)
        }
        return true;
    }
    // a biased token is its first entry's thread's: it knows where the entries lie
    __device__ __forceinline__ bool bias_value(int i, int& id, float& y) {
        id = i == b_at ? b_id : p.bias_id[i];
        const int before = i == b_at ? b_before : p.bias_id[i - 1];
        if (!real(id) || before >= id || !words.owns(id)) return false;
        unsigned* word = words.find(id);
        return value(id, TABLE ? 0x40000000u | (word ? atomicExch(word, 0u) : 0u) : atomicExch(word, 0u), i, y);
    }
    // (what is owned has been counted, so it is found)
    __device__ __forceinline__ bool text_value(int id, float& y) { return real(id) && words.owns(id) && value(id, atomicExch(words.find(id), 0u), -1, y); }

    // The mending, with a barrier in front, behind the counts.  `written` is called between the reading of the row and the first write: the copy is done
    // when it returns.  (A thread holds what it will write; where text or biases are more than that, everything is read and written behind the call.)
    template <typename F>
    __device__ __forceinline__ void mend(F written) {
        const bool all = w.b1 - w.b0 <= THREADS && w.len <= AHEAD * THREADS;
        int id;
        float y;
        if (!all) {
            written();
            for (int i = b_at; i < w.b1; i += THREADS)
                if (bias_value(i, id, y)) w.out[id] = y;
            __syncthreads();
            for (int first = 0; w.counts && first < w.len; first += AHEAD * THREADS) {
                fetch_text(first);
#pragma unroll
                for (int j = 0; j < AHEAD; ++j)
                    if (first + j * THREADS + tid < w.len && text_value(held[j], y)) w.out[held[j]] = y;
            }
            if (w.counts && tid == 0 && p.newest && text_value(w.newest, y)) w.out[w.newest] = y;
            return;
        }
        int bias_id = -1, newest_id = -1;
        float bias_y = 0.0f, newest_y = 0.0f, ys[AHEAD];
        if (b_at < w.b1 && bias_value(b_at, id, bias_y)) bias_id = id;
        if (w.counts) {
            if (TABLE && w.b0 < w.b1) __syncthreads();
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (!(j * THREADS + tid < w.len && text_value(held[j], ys[j]))) held[j] = -1;
            if (tid == 0 && p.newest && text_value(w.newest, newest_y)) newest_id = w.newest;
        }
        written();
        if (bias_id >= 0) w.out[bias_id] = bias_y;
        if (!w.counts) return;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (held[j] >= 0) w.out[held[j]] = ys[j];
        if (newest_id >= 0) w.out[newest_id] = newest_y;
    }
    // one CTA a row: the newest token into its place (which none of the row's CTAs reads)
    __device__ __forceinline__ void append() const {
        if (!w.history || !p.newest || tid != 0) return;
        if (w.newest >= 0 && w.newest < p.V && w.len < p.cap) w.history[w.len] = w.newest;
        else bad();
    }
};

constexpr int AL_TABLE_BITS = 14;      // the largest table: 128 KB

// Few rows: copy and mending of a range.
template <int THREADS, int LOADS, int VEC>
__global__ void __launch_bounds__(THREADS) adjust_logits_kernel(LogitsParams p) {
    constexpr int RANGE = THREADS * LOADS * VEC;
    __shared__ __align__(16) unsigned word_s[RANGE];
    pdl_launch();
    pdl_wait();
    const LogitsRow w(p, blockIdx.y);
    const int v0 = blockIdx.x * RANGE, v1 = min(p.V, v0 + RANGE);
    const bool marked = w.counts || w.b0 < w.b1;
    LogitsMend<THREADS, LogitsDense> m(p, w, LogitsDense{word_s, v0, v1});
    LogitsRange<THREADS, LOADS, VEC> range;
    if (marked) m.fetch();
    range.load(w, v0, v1);
    if (blockIdx.x == 0) m.append();
    if (marked) {
        m.words.template clear<THREADS>(RANGE);
        __syncthreads();
        m.count();
    }
    range.store(w, v0, v1);
    if (!marked) return;
    __syncthreads();
    m.mend([] {});
}

// Many rows: the copy ...
template <int THREADS, int LOADS, int VEC>
__global__ void __launch_bounds__(THREADS) copy_logits_kernel(LogitsParams p) {
    constexpr int RANGE = THREADS * LOADS * VEC;
    pdl_wait();
    pdl_launch();                                      // (the mending may count beside the copy: what it reads is there)
    const LogitsRow w(p, blockIdx.y);
    const int v0 = blockIdx.x * RANGE, v1 = min(p.V, v0 + RANGE);
    LogitsRange<THREADS, LOADS, VEC> range;
    range.load(w, v0, v1);
    range.store(w, v0, v1);
}

// ... and the mending.  `ahead`: the launch ahead is the copy's.  RANGE 0: a row's whole text in a table of 2^bits.
template <int THREADS, int RANGE>
__global__ void __launch_bounds__(THREADS) mend_logits_kernel(LogitsParams p, int ahead, int bits) {
    extern __shared__ __align__(16) unsigned mend_s[];
    pdl_launch();
    if (!ahead) pdl_wait();
    const LogitsRow w(p, blockIdx.y);
    const bool marked = w.counts || w.b0 < w.b1;
    auto work = [&](auto& m) {
        if (marked) {
            m.fetch();
            m.words.template clear<THREADS>(RANGE);
            __syncthreads();
            m.count();
        }
        auto written = [&]() { if (ahead) pdl_wait(); };
        if (!marked) written();
        else {
            __syncthreads();
            m.mend(written);
        }
        if (blockIdx.x == 0) m.append();
    };
    if constexpr (RANGE > 0) {
        const int v0 = blockIdx.x * RANGE;
        LogitsMend<THREADS, LogitsDense> m(p, w, LogitsDense{mend_s, v0, min(p.V, v0 + RANGE)});
        work(m);
    } else {
        LogitsMend<THREADS, LogitsTable> m(p, w, LogitsTable{(int*)mend_s, mend_s + (1 << bits), bits, (int)blockIdx.x, (int)gridDim.x});
        work(m);
    }
}

template <int THREADS, int LOADS, int VEC>
static int al_launch(const LogitsParams& p, int n, cudaStream_t stream) {
    constexpr int range = THREADS * LOADS * VEC;
    cudaError_t e = launch(adjust_logits_kernel<THREADS, LOADS, VEC>, dim3((unsigned)((p.V + range - 1) / range), (unsigned)n), dim3(THREADS), 0, stream, p);
    return e == cudaSuccess ? BG_OK : (int)e;
}

template <int THREADS, int LOADS, int VEC>
static int al_copy(const LogitsParams& p, int n, cudaStream_t stream) {
    constexpr int range = THREADS * LOADS * VEC;
    cudaError_t e = launch(copy_logits_kernel<THREADS, LOADS, VEC>, dim3((unsigned)((p.V + range - 1) / range), (unsigned)n), dim3(THREADS), 0, stream, p);
    return e == cudaSuccess ? BG_OK : (int)e;
}

template <int THREADS, int RANGE>
static int al_mend(const LogitsParams& p, int n, int ahead, cudaStream_t stream, int bits = 0, int parts = 1) {
    auto kern = mend_logits_kernel<THREADS, RANGE>;
    const size_t smem = RANGE ? (size_t)RANGE * 4 : (size_t)8 << bits;
    cudaError_t e = smem_limit(kern, RANGE ? smem : (size_t)8 << AL_TABLE_BITS);
    if (e != cudaSuccess) return (int)e;
    e = launch(kern, dim3((unsigned)(RANGE ? (p.V + RANGE - 1) / RANGE : parts), (unsigned)n), dim3(THREADS), smem, stream, p, ahead, bits);
    return e == cudaSuccess ? BG_OK : (int)e;
}

}  // namespace bg

using namespace bg;

// What a call hands over.  The host side fills the fields by name.
struct LogitsArgs {
    const float* x; float* out; int* history; const int* lengths; const int* prompts; const int* newest;
    const float* repetition; const float* frequency; const float* presence;
    const int* bias_id; const float* bias; const int* bias_row; const int* allowed; const int* allowed_row; unsigned* status;
    long long ldx, ldo;
    int n, V, cap, n_bias, words, masks;
};

// Bytes of what the host side mirrors field by field; it compares them when it loads the library.
extern "C" int bg_logits_bytes() { return (int)sizeof(LogitsArgs); }

// See the head of this file; `out` may be `x`.  A token outside [0, V), a row's biased tokens out of order, a full history and a mask that is not there set
// BG_STATUS_BAD_TOKEN and are passed over.  launched: how many kernels.
extern "C" int bg_adjust_logits(const LogitsArgs* args, int* launched, cudaStream_t stream) {
    const LogitsArgs& a = *args;
    *launched = 0;
    const int n = a.n, V = a.V, cap = a.cap;
    if (n <= 0) return BG_OK;
    if (V <= 0 || n > 65535 || a.ldx < V || a.ldo < V || (a.history && (!a.lengths || cap <= 0 || cap > 0x3ffffff0)) || (a.newest && !a.history)) return BG_ERR_SHAPE;
    if ((a.bias_id && (!a.bias || !a.bias_row || a.n_bias < 0)) || (a.allowed && (a.words < (V + 31) / 32 || a.masks <= 0))) return BG_ERR_SHAPE;
    if (V > 0x7fffffff - 65536) return BG_ERR_SHAPE;
    const LogitsParams p{a.x, a.ldx, a.out, a.ldo, V, a.history, cap, a.lengths, a.prompts, a.newest, a.repetition, a.frequency, a.presence, a.bias_id, a.bias,
                         a.bias_row, a.n_bias, (const unsigned*)a.allowed, a.words, a.allowed_row, a.masks, a.status};
    const bool pieces = a.ldx % 4 == 0 && a.ldo % 4 == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.out % 16 == 0;
    *launched = 1;
    // few rows: a CTA copies and mends a range
    const int sms = sm_count();
    if ((long long)n * ((V + 1023) / 1024) <= 2 * sms) return pieces ? al_launch<256, 1, 4>(p, n, stream) : al_launch<256, 4, 1>(p, n, stream);
    if ((long long)n * ((V + 2047) / 2048) <= 4 * sms) return pieces ? al_launch<256, 2, 4>(p, n, stream) : al_launch<256, 8, 1>(p, n, stream);
    const bool copies = a.x != a.out || a.allowed, mends = a.bias_id || ((a.repetition || a.frequency || a.presence) && a.history) || a.newest;
    *launched = copies + mends;
    int rc = BG_OK;
    if (copies) rc = pieces ? al_copy<256, 4, 4>(p, n, stream) : al_copy<256, 8, 1>(p, n, stream);
    if (rc != BG_OK || !mends) return rc;
    // texts that a table of AL_TABLE_BITS holds (by their room: the lengths are the device's); else ranges of the vocabulary
    int bits = 10, parts = 1;
    while (bits < AL_TABLE_BITS && (3LL << bits) < 4LL * (cap + 1)) ++bits;
    if ((3LL << bits) < 4LL * (cap + 1)) return al_mend<512, 16384>(p, n, copies, stream);
    while (parts < 4 && 2 * parts * n <= sms) parts *= 2;
    return al_mend<1024, 0>(p, n, copies, stream, bits, parts);
}
