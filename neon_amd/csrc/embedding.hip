// Embedding lookup with scaling, and the dense gradient of its table.
//
//   forward   out[j, :] = scale * W[ids[j], :]
//   gradient  dW = beta * dW + scale * G,  G[w, :] = sum of err[j, :] over the positions j with ids[j] == w
//
// Positions that hold the padding word, and words outside the table, give a
// zero row and no gradient; rows of G without a position are zero.  Both are
// bound by HBM traffic.  Every sum is taken in a fixed order (no floating-point
// atomics), in fp32, and rounded once.
//
// The gradient goes over the positions sorted by word:
//   1. lut_sort_kernel    256 workgroups; workgroup b owns the words with (word & 255) == b and puts
//                         their positions in word order, positions ascending within a word
//   2. lut_sum_kernel     a wave per 32 sorted positions and block of columns: adds error rows, stores
//                         words that begin and end inside, leaves partial sums of the others; further
//                         workgroups clear (or scale) the rows of absent words
//   3. lut_join_kernel    adds the partial sums of every word that crosses such a border
// A frequent word (a tenth of all positions in ordinary text) is spread over as
// many waves as it has runs of 32 positions.
#include "lm_ops.h"

namespace {

using lm::vec;

constexpr uint32_t NO_WORD = 0xFFFFFFFFu;

NEON_DEV bool in_table(uint32_t w, uint32_t vocab, uint32_t pad) { return w < vocab && w != pad; }

// ---------------------------------------------------------------------------
// forward, a position's values side by side: a group of 2^tpr_log threads per position
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void lut_rows_fprop_kernel(T* out, const T* W, const int32_t* ids, float scale, size_t count,
                                                             uint32_t embed, uint32_t vocab, uint32_t pad, size_t ld_w,
                                                             size_t ld_out, int tpr_log) {
    constexpr int V = vec<T>::V;
    const int tpr = 1 << tpr_log;
    const size_t j = (size_t)blockIdx.x * (256 >> tpr_log) + (threadIdx.x >> tpr_log);
    if (j >= count) return;
    const uint32_t w = (uint32_t)ids[j];
    const bool live = in_table(w, vocab, pad);
    const T* src = W + (size_t)(live ? w : 0) * ld_w;
    T* dst = out + j * ld_out;
    for (uint32_t c = (threadIdx.x & (tpr - 1)) * V; c < embed; c += tpr * V) {
        const int n = embed - c >= V ? V : (int)(embed - c);
        nh_raw<T, V> r;
        if (!live) r.zero();
        else if (n == V) r.load(src + c);
        else r.load_partial(src + c, n);
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int k = 0; k < V; ++k) o.set(k, live ? r.get(k) * scale : 0.0f);
        if (n == V) o.store(dst + c);
        else o.store_partial(dst + c, n);
    }
}

// forward, positions side by side: tiles of 128 positions and 128 bytes of columns, turned in LDS
constexpr int TURN_POS = 128;
template <typename T>
__global__ __launch_bounds__(256) void lut_cols_fprop_kernel(T* out, const T* W, const int32_t* ids, float scale, size_t count,
                                                             uint32_t embed, uint32_t vocab, uint32_t pad, size_t ld_w,
                                                             size_t ld_out) {
    constexpr int V = vec<T>::V, COLS = 8 * V, LD = COLS + 4 / (int)sizeof(T);
    __shared__ T tile[TURN_POS * LD];
    const uint32_t tiles_c = (uint32_t)((embed + COLS - 1) / COLS);
    const size_t j0 = (size_t)(blockIdx.x / tiles_c) * TURN_POS;
    const uint32_t c0 = (blockIdx.x % tiles_c) * COLS;
    {
        const uint32_t c = c0 + (threadIdx.x & 7) * V;
#pragma unroll
        for (int i = 0; i < TURN_POS / 32; ++i) {
            const int p = (threadIdx.x >> 3) + i * 32;
            const size_t j = j0 + p;
            const uint32_t w = j < count ? (uint32_t)ids[j] : NO_WORD;
            const bool live = in_table(w, vocab, pad) && c < embed;
            const T* src = W + (size_t)(live ? w : 0) * ld_w + c;
            nh_raw<T, V> r;
            if (!live) r.zero();
            else if (embed - c >= V) r.load(src);
            else r.load_partial(src, (int)(embed - c));
#pragma unroll
            for (int k = 0; k < V; ++k) tile[p * LD + (threadIdx.x & 7) * V + k] = (T)(live ? r.get(k) * scale : 0.0f);
        }
    }
    __syncthreads();
    constexpr int LP = TURN_POS / V;          // lanes along the positions of one output line
    const int p = (threadIdx.x % LP) * V;
    const size_t j = j0 + p;
    const int n = j >= count ? 0 : (count - j >= V ? V : (int)(count - j));
    if (n == 0) return;
    for (int e = threadIdx.x / LP; e < COLS && c0 + e < embed; e += 256 / LP) {
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int k = 0; k < V; ++k) o.set(k, (float)tile[(p + k) * LD + e]);
        T* dst = out + (size_t)(c0 + e) * ld_out + j;
        if (n == V) o.store(dst);
        else o.store_partial(dst, n);
    }
}

// ---------------------------------------------------------------------------
// sorting the positions
// ---------------------------------------------------------------------------
constexpr int GROUPS_LOG = 8, GROUPS = 1 << GROUPS_LOG;      // workgroups of the sort = classes of words
constexpr int SORT_T = 1024, SORT_W = SORT_T / 64;

struct SortArgs {
    const int32_t* ids;
    uint2* a;             // (word, position), `count` entries each
    uint2* b;
    uint32_t* present;    // a bit per word: GROUPS runs of `words_per` 32-bit words
    uint32_t* total;      // number of sorted positions
    uint32_t count, vocab, pad, words_per;
    int passes;           // of 8 bits over word >> GROUPS_LOG
};

// sum of v over the workgroup, and over the threads before this one's wave
NEON_DEV uint32_t wave_sum(uint32_t v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += (uint32_t)__shfl_xor((int)v, d);
    return v;
}

__global__ __launch_bounds__(SORT_T) void lut_sort_kernel(SortArgs s) {
    __shared__ uint32_t w_match[SORT_W], w_lower[SORT_W];
    __shared__ uint32_t hist[SORT_W][256];
    __shared__ uint32_t scan[256];
    const uint32_t cls = blockIdx.x;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned long long below = (1ull << lane) - 1ull;
    // a wave looks at a contiguous run of the ids, 4 per lane and step
    const uint32_t steps = (s.count + 4 * SORT_T - 1) / (4 * SORT_T);
    const uint32_t first = (uint32_t)wave * steps * 256;

    uint32_t match = 0, lower = 0;
    for (uint32_t i = 0; i < steps; ++i) {
        const uint32_t p = first + i * 256 + lane * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w = p + k < s.count ? (uint32_t)s.ids[p + k] : NO_WORD;
            const bool live = in_table(w, s.vocab, s.pad);
            const uint32_t c = w & (GROUPS - 1);
            match += live && c == cls;
            lower += live && c < cls;
        }
    }
    match = wave_sum(match);
    lower = wave_sum(lower);
    if (lane == 0) {
        w_match[wave] = match;
        w_lower[wave] = lower;
    }
    // this class's part of the presence bits, cleared
    uint32_t* bits = s.present + (size_t)cls * s.words_per;
    for (uint32_t i = t; i < s.words_per; i += SORT_T) bits[i] = 0;
    __syncthreads();
    uint32_t start = 0, mine = 0, n = 0;
#pragma unroll
    for (int w = 0; w < SORT_W; ++w) {
        start += w_lower[w];
        mine += w < wave ? w_match[w] : 0;
        n += w_match[w];
    }
    if (cls == GROUPS - 1 && t == 0) *s.total = start + n;
    if (n == 0) return;

    // the class's positions, ascending
    uint2* from = s.a + start;
    uint2* to = s.b + start;
    uint32_t at = mine;
    for (uint32_t i = 0; i < steps; ++i) {
        const uint32_t p = first + i * 256 + lane * 4;
        uint32_t w[4];
        unsigned long long m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[k] = p + k < s.count ? (uint32_t)s.ids[p + k] : NO_WORD;
            m[k] = __ballot(in_table(w[k], s.vocab, s.pad) && (w[k] & (GROUPS - 1)) == cls);
        }
        if ((m[0] | m[1] | m[2] | m[3]) == 0) continue;
        uint32_t o = at;
#pragma unroll
        for (int k = 0; k < 4; ++k) o += __popcll(m[k] & below);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if ((m[k] >> lane) & 1ull) {
                from[o++] = make_uint2(w[k], p + k);
                const uint32_t local = w[k] >> GROUPS_LOG;
                atomicOr(&bits[local >> 5], 1u << (local & 31));
            }
            at += __popcll(m[k]);
        }
    }
    __syncthreads();

    // least significant digit first, 8 bits a pass, stable: a wave owns a contiguous run of the entries
    const uint32_t run = (n + SORT_T - 1) / SORT_T * 64;      // entries per wave
    const uint32_t e0 = (uint32_t)wave * run < n ? (uint32_t)wave * run : n;
    const uint32_t e1 = e0 + run < n ? e0 + run : n;
    for (int pass = 0; pass < s.passes; ++pass) {
        const int shift = GROUPS_LOG + 8 * pass;
#pragma unroll
        for (int i = 0; i < 4; ++i) hist[wave][lane + 64 * i] = 0;
        __syncthreads();
        for (uint32_t e = e0 + lane; e < e1; e += 64) atomicAdd(&hist[wave][(from[e].x >> shift) & 255u], 1u);
        __syncthreads();
        // offsets in the order (digit, wave)
        uint32_t sum = 0;
        if (t < 256) {
#pragma unroll
            for (int w = 0; w < SORT_W; ++w) {
                const uint32_t h = hist[w][t];
                hist[w][t] = sum;
                sum += h;
            }
            scan[t] = sum;
        }
        __syncthreads();
        if (wave == 0) {
            uint32_t v[4], tot = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = tot;
                tot += scan[lane * 4 + i];
            }
            uint32_t inc = tot;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = (uint32_t)__shfl_up((int)inc, d);
                inc += lane >= d ? up : 0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) scan[lane * 4 + i] = inc - tot + v[i];
        }
        __syncthreads();
        for (uint32_t base = e0; base < e1; base += 64) {
            const uint32_t e = base + lane;
            const bool on = e < e1;
            const uint2 item = on ? from[e] : make_uint2(0, 0);
            const uint32_t digit = (item.x >> shift) & 255u;
            unsigned long long same = __ballot(on);
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const unsigned long long set = __ballot((digit >> b) & 1u);
                same &= ((digit >> b) & 1u) ? set : ~set;
            }
            uint32_t o = 0;
            if (on) o = scan[digit] + hist[wave][digit] + __popcll(same & below);
            // every lane has read its counter before the first lane of each digit moves it on
            __builtin_amdgcn_wave_barrier();
            if (on) {
                to[o] = item;
                if ((same & below) == 0) hist[wave][digit] += __popcll(same);
            }
            __builtin_amdgcn_wave_barrier();
        }
        uint2* swap = from;
        from = to;
        to = swap;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// adding up
// ---------------------------------------------------------------------------
constexpr int RUN = 32;          // sorted positions per wave

struct SumArgs {
    void* dW;
    const void* err;
    const uint2* sorted;
    const uint32_t* present;
    const uint32_t* total;
    float* part;                 // [run][head, tail][embed]
    float scale, beta;
    uint32_t embed, vocab, words_per, tiles;
    uint32_t sum_blocks;         // workgroups that add; the others clear
    size_t ld_dw, ld_err;
};

template <typename T, int V> NEON_DEV void put_row(T* dst, const float (&acc)[V], int n, float scale, float beta) {
    nh_out<T, V> o;
    o.clear();
    if (beta != 0.0f) {
        nh_raw<T, V> old;
        if (n == V) old.load(dst);
        else old.load_partial(dst, n);
#pragma unroll
        for (int k = 0; k < V; ++k) o.set(k, __builtin_fmaf(beta, old.get(k), scale * acc[k]));
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) o.set(k, scale * acc[k]);
    }
    if (n == V) o.store(dst);
    else o.store_partial(dst, n);
}

constexpr int CLEAR_ROWS = 32;      // rows of the table per clearing workgroup

template <typename T> NEON_DEV void clear_rows(const SumArgs& a, uint32_t block) {
    constexpr int V = vec<T>::V;
    const int lane = threadIdx.x & 63;
    for (uint32_t i = threadIdx.x >> 6; i < CLEAR_ROWS; i += 4) {
        const size_t w = (size_t)block * CLEAR_ROWS + i;
        if (w >= a.vocab) return;
        const uint32_t local = (uint32_t)w >> GROUPS_LOG;
        if ((a.present[(size_t)(w & (GROUPS - 1)) * a.words_per + (local >> 5)] >> (local & 31)) & 1u) continue;
        T* row = (T*)a.dW + w * a.ld_dw;
        const float zero[V] = {};
        for (uint32_t c = lane * V; c < a.embed; c += 64 * V)
            put_row<T, V>(row + c, zero, a.embed - c >= V ? V : (int)(a.embed - c), 0.0f, a.beta);
    }
}

template <typename T> __global__ __launch_bounds__(256) void lut_sum_kernel(SumArgs a) {
    constexpr int V = vec<T>::V;
    if (blockIdx.x >= a.sum_blocks) {
        clear_rows<T>(a, blockIdx.x - a.sum_blocks);
        return;
    }
    const int lane = threadIdx.x & 63;
    const size_t id = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const size_t run = id / a.tiles;
    const uint32_t c = ((uint32_t)(id % a.tiles) * 64 + lane) * V;
    const uint32_t total = *a.total;
    const size_t s0 = run * RUN;
    if (s0 >= total) return;
    const int len = total - s0 < RUN ? (int)(total - s0) : RUN;
    const int n = c >= a.embed ? 0 : (a.embed - c >= V ? V : (int)(a.embed - c));
    const T* err = (const T*)a.err + c;
    // lane i holds entry i; lane 32 the word before the run, lane 33 the word after it
    uint2 item = make_uint2(NO_WORD, 0);
    if (lane < len) item = a.sorted[s0 + lane];
    else if (lane == 32 && s0 > 0) item = a.sorted[s0 - 1];
    else if (lane == 33 && s0 + len < total) item = a.sorted[s0 + len];
    const uint32_t before = (uint32_t)__builtin_amdgcn_readlane((int)item.x, 32);
    const uint32_t after = (uint32_t)__builtin_amdgcn_readlane((int)item.x, 33);
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    bool head = (uint32_t)__builtin_amdgcn_readlane((int)item.x, 0) == before;     // the word began in an earlier run
    constexpr int AHEAD = 8;
    for (int i0 = 0; i0 < len; i0 += AHEAD) {
        nh_raw<T, V> r[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int e = i0 + i < len ? i0 + i : len - 1;
            const uint32_t pos = (uint32_t)__builtin_amdgcn_readlane((int)item.y, e);
            if (n == V) r[i].load(err + (size_t)pos * a.ld_err);
            else if (n > 0) r[i].load_partial(err + (size_t)pos * a.ld_err, n);
            else r[i].zero();
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (i0 + i >= len) break;
            const int e = i0 + i;
            const uint32_t word = (uint32_t)__builtin_amdgcn_readlane((int)item.x, e);
            const uint32_t next = e + 1 < len ? (uint32_t)__builtin_amdgcn_readlane((int)item.x, e + 1) : after;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += r[i].get(k);
            const bool last = e + 1 == len;
            if (next != word || last) {
                const bool goes_on = last && next == word;
                if (n > 0) {
                    if (head || goes_on) {
                        float* p = a.part + (run * 2 + (head ? 0 : 1)) * a.embed + c;
#pragma unroll
                        for (int k = 0; k < V; ++k)
                            if (k < n) p[k] = acc[k];
                    } else {
                        put_row<T, V>((T*)a.dW + (size_t)word * a.ld_dw + c, acc, n, a.scale, a.beta);
                    }
                }
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] = 0.0f;
                head = false;
            }
        }
    }
}

// A workgroup per run and 256 columns.  Where a word begins in the run and goes
// on behind it: tail of this run + heads of the following ones, the runs dealt
// to the waves in contiguous shares and the shares joined in order.
constexpr int JOIN_T = 512, JOIN_W = JOIN_T / 64;
template <typename T> __global__ __launch_bounds__(JOIN_T) void lut_join_kernel(SumArgs a) {
    __shared__ float share[JOIN_W][256];
    const uint32_t total = *a.total;
    const uint32_t tiles = (a.embed + 255) / 256;
    const size_t run = blockIdx.x / tiles;
    const uint32_t c = (blockIdx.x % tiles) * 256 + (threadIdx.x & 63) * 4;
    const size_t s0 = run * RUN;
    if (s0 + RUN >= total) return;                             // nothing behind this run
    const uint32_t word = a.sorted[s0 + RUN - 1].x;
    if (a.sorted[s0 + RUN].x != word) return;                  // no word crosses its end
    if (s0 > 0 && a.sorted[s0 - 1].x == word && a.sorted[s0].x == word) return;      // it began before this run
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // the last run with this word: the first border (run k begins at k * RUN) whose word differs
    size_t last = run + 1;
    for (;;) {
        const size_t k = last + 1 + lane;
        const bool same = k * RUN < total && a.sorted[k * RUN].x == word;
        const unsigned long long m = __ballot(same);
        if (m == ~0ull) {
            last += 64;
            continue;
        }
        last += __builtin_ctzll(~m);
        break;
    }
    const int n = c >= a.embed ? 0 : (a.embed - c >= 4 ? 4 : (int)(a.embed - c));
    const size_t heads = last - run;                           // runs run + 1 .. last
    const size_t per = (heads + JOIN_W - 1) / JOIN_W;
    const size_t h0 = run + 1 + (size_t)wave * per, h1 = h0 + per < last + 1 ? h0 + per : last + 1;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (wave == 0)
        for (int k = 0; k < n; ++k) acc[k] = a.part[(run * 2 + 1) * a.embed + c + k];
#pragma unroll 4
    for (size_t h = h0; h < h1; ++h) {
        const float* p = a.part + h * 2 * a.embed + c;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (n == 4) nh_load_vec<float, 4>(p, v);
        else
            for (int k = 0; k < n; ++k) v[k] = p[k];
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] += v[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) share[wave][lane * 4 + k] = acc[k];
    __syncthreads();
    if (wave == 0 && n > 0) {
#pragma unroll
        for (int w = 1; w < JOIN_W; ++w)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] += share[w][lane * 4 + k];
        put_row<T, 4>((T*)a.dW + (size_t)word * a.ld_dw + c, acc, n, a.scale, a.beta);
    }
}

// ---------------------------------------------------------------------------
// workspace of the gradient
// ---------------------------------------------------------------------------
struct Layout {
    size_t a, b, present, total, part, turned, bytes;
    uint32_t words_per;
};

Layout layout(int dtype, int axis, size_t count, size_t embed, size_t vocab) {
    Layout l;
    size_t at = 0;
    const auto take = [&at](size_t bytes) {
        const size_t here = at;
        at += lm::align256(bytes);
        return here;
    };
    l.words_per = (uint32_t)lm::ceil_div(lm::ceil_div(vocab, GROUPS), 32);
    l.a = take(count * sizeof(uint2));
    l.b = take(count * sizeof(uint2));
    l.present = take((size_t)GROUPS * l.words_per * 4);
    l.total = take(4);
    l.part = take(lm::ceil_div(count, RUN) * 2 * embed * sizeof(float));
    l.turned = take(axis == 0 ? count * embed * lm::item_bytes(dtype) : 0);
    l.bytes = at;
    return l;
}

int check(const char* who, int dtype, int axis, size_t count, size_t embed, size_t vocab, size_t ld_table, size_t ld_values) {
    if (!lm::known_dtype(dtype)) return lm::refuse(who, "unknown storage type");
    if (axis != 0 && axis != 1) return lm::refuse(who, "axis is 0 or 1");
    if (embed == 0 || embed > 0x7FFFFFF) return lm::refuse(who, "between 1 and 2^27 - 1 columns");
    if (vocab == 0 || vocab > 0x7FFFFFFF) return lm::refuse(who, "between 1 and 2^31 - 1 words");
    if (count > 0x7FFFFFFF) return lm::refuse(who, "more than 2^31 - 1 positions");
    if (vocab > 1 && ld_table < embed) return lm::refuse(who, "leading dimension of the table shorter than a row");
    const size_t len = axis == 1 ? embed : count, lines = axis == 1 ? count : embed;
    if (lines > 1 && ld_values < len) return lm::refuse(who, "leading dimension shorter than a line");
    return 0;
}

uint32_t pad_word(int64_t pad_idx) { return pad_idx >= 0 && pad_idx <= 0x7FFFFFFF ? (uint32_t)pad_idx : NO_WORD; }

}  // namespace

extern "C" {

int nh_embed_fprop(void* out, const void* W, const int32_t* ids, float scale, int dtype, int axis, size_t positions,
                   size_t embed, size_t vocab, size_t ld_w, size_t ld_out, int64_t pad_idx, void* stream) {
    const char* who = "nh_embed_fprop";
    if (int rc = check(who, dtype, axis, positions, embed, vocab, ld_w, ld_out)) return rc;
    if (positions == 0) return 0;
    if (!out || !W || !ids) return lm::refuse(who, "null pointer");
    if (!nh_internal_ready()) return nh_internal_fail(NH_ENOTINIT, "nh_init has not been called");
    lm::OnDevice here;
    const hipStream_t s = (hipStream_t)stream;
    const uint32_t pad = pad_word(pad_idx);
    return lm::by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr size_t V = vec<T>::V;
        if (axis == 1) {
            int log = 0;
            while (log < 8 && ((size_t)V << log) < embed) ++log;
            const size_t blocks = lm::ceil_div(positions, (size_t)256 >> log);
            if (blocks > lm::MAX_BLOCKS) return lm::refuse(who, "too large for one launch");
            hipLaunchKernelGGL((lut_rows_fprop_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, (T*)out, (const T*)W, ids,
                               scale, positions, (uint32_t)embed, (uint32_t)vocab, pad, ld_w, ld_out, log);
        } else {
            const size_t blocks = lm::ceil_div(positions, TURN_POS) * lm::ceil_div(embed, 8 * V);
            if (blocks > lm::MAX_BLOCKS) return lm::refuse(who, "too large for one launch");
            hipLaunchKernelGGL((lut_cols_fprop_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, (T*)out, (const T*)W, ids,
                               scale, positions, (uint32_t)embed, (uint32_t)vocab, pad, ld_w, ld_out);
        }
        return lm::launched(who);
    });
}

size_t nh_embed_update_workspace_bytes(int dtype, int axis, size_t positions, size_t embed, size_t vocab) {
    if (check("nh_embed_update_workspace_bytes", dtype, axis, positions, embed, vocab, embed, axis == 1 ? embed : positions)) return 0;
    return layout(dtype, axis, positions, embed, vocab).bytes;
}

int nh_embed_update(void* dW, const void* err, const int32_t* ids, float scale, float beta, int dtype, int axis,
                    size_t positions, size_t embed, size_t vocab, size_t ld_dw, size_t ld_err, int64_t pad_idx, void* workspace,
                    size_t workspace_bytes, void* stream) {
    const char* who = "nh_embed_update";
    if (int rc = check(who, dtype, axis, positions, embed, vocab, ld_dw, ld_err)) return rc;
    if (!dW || (positions && (!err || !ids))) return lm::refuse(who, "null pointer");
    const Layout l = layout(dtype, axis, positions, embed, vocab);
    if (!workspace || workspace_bytes < l.bytes) return lm::refuse(who, "workspace smaller than nh_embed_update_workspace_bytes");
    if (!nh_internal_ready()) return nh_internal_fail(NH_ENOTINIT, "nh_init has not been called");
    lm::OnDevice here;
    const hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    return lm::by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr size_t V = vec<T>::V;
        SortArgs q = {};
        q.ids = ids;
        q.a = (uint2*)(ws + l.a);
        q.b = (uint2*)(ws + l.b);
        q.present = (uint32_t*)(ws + l.present);
        q.total = (uint32_t*)(ws + l.total);
        q.count = (uint32_t)positions;
        q.vocab = (uint32_t)vocab;
        q.pad = pad_word(pad_idx);
        q.words_per = l.words_per;
        for (size_t rest = (vocab - 1) >> GROUPS_LOG; rest; rest >>= 8) ++q.passes;
        hipLaunchKernelGGL(lut_sort_kernel, dim3(GROUPS), dim3(SORT_T), 0, s, q);
        SumArgs a = {};
        a.dW = dW;
        a.err = err;
        a.ld_err = ld_err;
        if (axis == 0 && positions) {
            // (embed, positions) -> (positions, embed)
            const uint32_t shape[2] = {(uint32_t)positions, (uint32_t)embed};
            const int64_t to[2] = {(int64_t)embed, 1}, from[2] = {1, (int64_t)ld_err};
            if (int rc = nh_copy_transpose(ws + l.turned, err, sizeof(T), 2, shape, to, from, stream)) return rc;
            a.err = ws + l.turned;
            a.ld_err = embed;
        }
        a.sorted = q.passes & 1 ? q.b : q.a;
        a.present = q.present;
        a.total = q.total;
        a.part = (float*)(ws + l.part);
        a.scale = scale;
        a.beta = beta;
        a.embed = (uint32_t)embed;
        a.vocab = (uint32_t)vocab;
        a.words_per = l.words_per;
        a.ld_dw = ld_dw;
        a.tiles = (uint32_t)lm::ceil_div(embed, 64 * V);
        const size_t runs = lm::ceil_div(positions, RUN);
        const size_t adding = lm::ceil_div(runs * a.tiles, 4), joining = runs * lm::ceil_div(embed, 256);
        const size_t clearing = beta == 1.0f ? 0 : lm::ceil_div(vocab, CLEAR_ROWS);
        if (adding + clearing > lm::MAX_BLOCKS || joining > lm::MAX_BLOCKS) return lm::refuse(who, "too large for one launch");
        a.sum_blocks = (uint32_t)adding;
        if (adding + clearing)
            hipLaunchKernelGGL((lut_sum_kernel<T>), dim3((unsigned)(adding + clearing)), dim3(256), 0, s, a);
        if (runs > 1) hipLaunchKernelGGL((lut_join_kernel<T>), dim3((unsigned)joining), dim3(JOIN_T), 0, s, a);
        return lm::launched(who);
    });
}

}  // extern "C"
