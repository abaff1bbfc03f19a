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
//   1. lut_split_kernel   a workgroup per 4096 positions puts them in the order of the 256 classes
//                         word & 255, and leaves where each class begins; further workgroups turn
//                         errors in the (embed, positions) layout around
//   2. lut_class_kernel   a workgroup per class collects its share of every slice and sorts it by
//                         word, positions ascending within a word
//   3. lut_sum_kernel     a wave per run of sorted positions and block of columns: adds error rows,
//                         stores words that begin and end inside, leaves partial sums of the others;
//                         further workgroups clear (or scale) the rows of absent words
//   4. lut_join_kernel    adds the partial sums of every word that crosses the end of a run
// A frequent word (a tenth of all positions in ordinary text) is spread over as
// many waves as it fills runs.  32768 positions, 50000 x 1024 bf16: 6 + 8 + 36 + 6
// us, of which 31 us are the bytes (the errors once, the table once); 1 and 2 and 4
// wait for memory a few times in a row, whatever they move.
#include <type_traits>

#include "lm_ops.h"

namespace {

using lm::vec;

constexpr uint32_t NO_WORD = 0xFFFFFFFFu;

NEON_DEV bool in_table(uint32_t w, uint32_t vocab, uint32_t pad) { return w < vocab && w != pad; }

// ---------------------------------------------------------------------------
// forward, a position's values side by side: a group of 2^tpr_log threads per
// position.  Bound by HBM and the caches that hold the frequent rows: 16384 positions
// x 1024 fp16 of 32000 words 10 us (67 MB read and written, 6.5 TB/s); 65536 x 300 fp32 27 us (157 MB, 5.8 TB/s).
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
// (16384 positions x 1024 fp16: 12 us, 67 MB, 5.6 TB/s)
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
constexpr int CLASS_LOG = 8, CLASSES = 1 << CLASS_LOG;
constexpr int SORT_T = 1024, SORT_W = SORT_T / 64;
constexpr int LOOKS = 4, SLICE = LOOKS * SORT_T;     // positions per workgroup of the split
constexpr uint32_t IN_LDS = 8192;    // entries of a class that are sorted without leaving the CU (half as many
                                     // where words take more than one pass)

struct SortArgs {
    const int32_t* ids;
    uint2* split;         // (word, position): slices of SLICE entries, each in class order
    uint32_t* table;      // [slice][CLASSES + 1]: where each class begins in the slice
    uint2* scratch;       // sorting space of classes that do not fit the LDS
    uint2* sorted;        // the entries, by class and word
    uint32_t* present;    // a bit per word: CLASSES runs of `words_per` 32-bit words
    uint32_t* total;      // number of sorted positions; behind it the lengths of lut_join_kernel's two lists
    uint32_t count, slices, vocab, pad, words_per;
    int passes;           // of 8 bits over word >> CLASS_LOG
};

NEON_DEV uint32_t wave_sum(uint32_t v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += (uint32_t)__shfl_xor((int)v, d);
    return v;
}
NEON_DEV uint32_t wave_scan(uint32_t v) {      // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t up = (uint32_t)__shfl_up((int)v, d);
        v += lane >= d ? up : 0;
    }
    return v;
}
// lanes of the wave that are on and have this lane's digit of 8 bits
NEON_DEV unsigned long long alike(bool on, uint32_t digit) {
    unsigned long long same = __ballot(on);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const unsigned long long set = __ballot((digit >> b) & 1u);
        same &= ((digit >> b) & 1u) ? set : ~set;
    }
    return same;
}

// Counters of a counting sort over 8 bits: a wave has its own 256 and owns a
// contiguous run of the entries, so it counts without atomics -- only the first
// lane of each digit adds (a word of a tenth of all positions would line up
// atomics behind one another).
struct Digits {
    uint32_t hist[SORT_W][256];
    uint32_t scan[256];
};
// Counters -> offsets in the order (digit, wave); every thread of the workgroup
// calls it.  With `bits`, a bit for every digit that occurs goes there.
NEON_DEV void offsets(Digits& m, uint32_t* bits, uint32_t bit_words) {
    const int t = threadIdx.x, lane = t & 63;
    __syncthreads();
    if (t < 256) {
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < SORT_W; ++w) {
            const uint32_t h = m.hist[w][t];
            m.hist[w][t] = sum;
            sum += h;
        }
        m.scan[t] = sum;
        const unsigned long long occurs = __ballot(sum > 0);
        const uint32_t word = (uint32_t)(t >> 6) * 2 + lane;
        if (bits && lane < 2 && word < bit_words) bits[word] = (uint32_t)(occurs >> (32 * lane));
    }
    __syncthreads();
    if (t < 64) {
        uint32_t v[4], tot = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = tot;
            tot += m.scan[lane * 4 + i];
        }
        const uint32_t before = wave_scan(tot) - tot;
#pragma unroll
        for (int i = 0; i < 4; ++i) m.scan[lane * 4 + i] = before + v[i];
    }
    __syncthreads();
}

// (embed, positions) -> (positions, embed): tiles of 64 columns
struct TurnArgs {
    const void* from;
    void* to;
    uint32_t count, embed, tiles_e;
    size_t ld;
};
template <typename T> struct turn {
    static constexpr int V = vec<T>::V, E = 64, P = SORT_T * V / E, LD = P + 4 / (int)sizeof(T);
};
template <typename T> NEON_DEV void turn_tile(const TurnArgs& a, uint32_t block, T* tile) {
    constexpr int V = turn<T>::V, E = turn<T>::E, P = turn<T>::P, LD = turn<T>::LD;
    const uint32_t p0 = block / a.tiles_e * P, e0 = block % a.tiles_e * E;
    {
        const uint32_t e = e0 + threadIdx.x / (P / V), p = p0 + threadIdx.x % (P / V) * V;
        if (e < a.embed && p < a.count) {
            const T* src = (const T*)a.from + (size_t)e * a.ld + p;
            nh_raw<T, V> r;
            if (a.count - p >= V) r.load(src);
            else r.load_partial(src, (int)(a.count - p));
#pragma unroll
            for (int k = 0; k < V; ++k) tile[(e - e0) * LD + (p - p0) + k] = nh_store_cvt<T>::f(r.get(k));
        }
    }
    __syncthreads();
    const uint32_t e = e0 + threadIdx.x % (E / V) * V, p = p0 + threadIdx.x / (E / V);
    if (e >= a.embed || p >= a.count) return;
    nh_out<T, V> o;
    o.clear();
#pragma unroll
    for (int k = 0; k < V; ++k) o.set(k, (float)tile[(e - e0 + k) * LD + (p - p0)]);
    T* dst = (T*)a.to + (size_t)p * a.embed + e;
    if (a.embed - e >= V) o.store(dst);
    else o.store_partial(dst, (int)(a.embed - e));
}

// The splitting workgroups wait for memory most of their time, the turning ones
// move data, and neither needs the other.
template <typename T> __global__ __launch_bounds__(SORT_T) void lut_split_kernel(SortArgs s, TurnArgs turned) {
    __shared__ union Space {
        Digits m;
        uint8_t tile[sizeof(T) * turn<T>::E * turn<T>::LD];
        __device__ Space() {}
    } space;
    if (blockIdx.x >= s.slices) {
        turn_tile<T>(turned, blockIdx.x - s.slices, reinterpret_cast<T*>(space.tile));
        return;
    }
    Digits& m = space.m;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned long long below = (1ull << lane) - 1ull;
    const uint32_t first = blockIdx.x * SLICE + wave * (SLICE / SORT_W) + lane;
    uint32_t w[LOOKS];
    unsigned long long same[LOOKS];
    bool on[LOOKS];
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) w[i] = first + i * 64 < s.count ? (uint32_t)s.ids[first + i * 64] : NO_WORD;
#pragma unroll
    for (int i = 0; i < 4; ++i) m.hist[wave][lane + 64 * i] = 0;
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
        on[i] = in_table(w[i], s.vocab, s.pad);
        same[i] = alike(on[i], w[i] & (CLASSES - 1));
        if (on[i] && (same[i] & below) == 0) m.hist[wave][w[i] & (CLASSES - 1)] += __popcll(same[i]);
    }
    offsets(m, nullptr, 0);
    uint32_t* table = s.table + (size_t)blockIdx.x * (CLASSES + 1);
    if (t < CLASSES) table[t] = m.scan[t];
    uint2* out = s.split + (size_t)blockIdx.x * SLICE;
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
        const uint32_t c = w[i] & (CLASSES - 1);
        uint32_t o = 0;
        if (on[i]) o = m.scan[c] + m.hist[wave][c] + __popcll(same[i] & below);
        // every lane has read its counter before the first lane of each class moves it on
        __builtin_amdgcn_wave_barrier();
        if (on[i]) {
            out[o] = make_uint2(w[i], first + i * 64);
            if ((same[i] & below) == 0) m.hist[wave][c] += __popcll(same[i]);
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // the last wave's counter of the last class now stands at the class's size
    if (t == 0) table[CLASSES] = m.scan[CLASSES - 1] + m.hist[SORT_W - 1][CLASSES - 1];
}

// One stable pass over 8 bits of the words: from[0, n) -> to[0, n).  Where these
// bits and the class are the whole word, `bits` gets the words that occur.
NEON_DEV void sort_pass(Digits& m, const uint2* from, uint2* to, uint32_t n, int shift, uint32_t* bits, uint32_t bit_words) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned long long below = (1ull << lane) - 1ull;
    const uint32_t run = (n + SORT_T - 1) / SORT_T * 64;
    const uint32_t e0 = (uint32_t)wave * run < n ? (uint32_t)wave * run : n;
    const uint32_t e1 = e0 + run < n ? e0 + run : n;
#pragma unroll
    for (int i = 0; i < 4; ++i) m.hist[wave][lane + 64 * i] = 0;
    for (uint32_t base = e0; base < e1; base += 64) {
        const bool on = base + lane < e1;
        const uint32_t digit = on ? (from[base + lane].x >> shift) & 255u : 0;
        const unsigned long long same = alike(on, digit);
        if (on && (same & below) == 0) m.hist[wave][digit] += __popcll(same);
    }
    offsets(m, bits, bit_words);
    for (uint32_t base = e0; base < e1; base += 64) {
        const bool on = base + lane < e1;
        const uint2 item = on ? from[base + lane] : make_uint2(0, 0);
        const uint32_t digit = (item.x >> shift) & 255u;
        const unsigned long long same = alike(on, digit);
        uint32_t o = 0;
        if (on) o = m.scan[digit] + m.hist[wave][digit] + __popcll(same & below);
        __builtin_amdgcn_wave_barrier();      // (as in the split)
        if (on) {
            to[o] = item;
            if ((same & below) == 0) m.hist[wave][digit] += __popcll(same);
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
}

__global__ __launch_bounds__(SORT_T) void lut_class_kernel(SortArgs s) {
    __shared__ Digits m;
    __shared__ uint2 lds[IN_LDS];
    __shared__ uint32_t w_len[SORT_W], w_low[SORT_W];
    __shared__ uint4 piece[SORT_T];           // a slice's share: where it begins there, its length, where it goes
    const uint32_t cls = blockIdx.x;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // where the class begins in a slice, and how much of the slice it is
    const auto share = [&](uint32_t slice) {
        if (slice >= s.slices) return make_uint2(0, 0);
        const uint32_t* p = s.table + (size_t)slice * (CLASSES + 1) + cls;
        const uint32_t b = p[0];
        return make_uint2(b, p[1] - b);
    };
    const uint2 mine = share(t);
    uint32_t low = mine.x, len = mine.y;
    for (uint32_t i = t + SORT_T; i < s.slices; i += SORT_T) {
        const uint2 more = share(i);
        low += more.x;
        len += more.y;
    }
    low = wave_sum(low);
    len = wave_sum(len);
    if (lane == 0) {
        w_len[wave] = len;
        w_low[wave] = low;
    }
    uint32_t* bits = s.present + (size_t)cls * s.words_per;
    if (s.passes != 1)
        for (uint32_t i = t; i < s.words_per; i += SORT_T) bits[i] = 0;
    __syncthreads();
    uint32_t start = 0, n = 0;
#pragma unroll
    for (int v = 0; v < SORT_W; ++v) {
        start += w_low[v];
        n += w_len[v];
    }
    if (cls == CLASSES - 1 && t == 0) {
        s.total[0] = start + n;
        s.total[1] = s.total[2] = 0;
    }
    if (n == 0) {
        if (s.passes == 1 && t < s.words_per) bits[t] = 0;
        return;
    }

    // the class's positions, ascending
    uint2* const out = s.sorted + start;
    const bool local = n <= (s.passes > 1 ? IN_LDS / 2 : IN_LDS);
    uint2* from = s.passes == 0 ? out : local ? lds : s.passes & 1 ? s.scratch + start : out;
    uint2* to = local ? lds + IN_LDS / 2 : s.passes & 1 ? out : s.scratch + start;
    uint32_t done = 0;
    for (uint32_t i0 = 0; i0 < s.slices; i0 += SORT_T) {
        const uint2 sh = i0 ? share(i0 + t) : mine;
        uint32_t at = wave_scan(sh.y);
        __syncthreads();                       // (w_len and piece of the turn before have been read)
        if (lane == 63) w_len[wave] = at;
        __syncthreads();
        at += done - sh.y;
        for (int v = 0; v < SORT_W; ++v) {
            at += v < wave ? w_len[v] : 0;
            done += w_len[v];
        }
        piece[t] = make_uint4(sh.x, sh.y, at, 0);
        __syncthreads();
        const uint32_t here = s.slices - i0 < SORT_T ? s.slices - i0 : SORT_T;
        for (uint32_t k = wave; k < here; k += SORT_W) {
            const uint4 pc = piece[k];
            const uint2* src = s.split + (size_t)(i0 + k) * SLICE + pc.x;
            for (uint32_t e = lane; e < pc.y; e += 64) from[pc.z + e] = src[e];
        }
    }
    __syncthreads();
    // least significant digit first; the last pass ends in `out`
    for (int pass = 0; pass < s.passes; ++pass) {
        uint2* const dst = pass + 1 == s.passes ? out : to;
        sort_pass(m, from, dst, n, CLASS_LOG + 8 * pass, s.passes == 1 ? bits : nullptr, s.words_per);
        to = from;
        from = dst;
    }
    if (s.passes == 1) return;
    // the words that occur
    for (uint32_t e = t; e < n; e += SORT_T) {
        const uint32_t word = out[e].x;
        if (e == 0 || out[e - 1].x != word) {
            const uint32_t k = word >> CLASS_LOG;
            atomicOr(&bits[k >> 5], 1u << (k & 31));
        }
    }
}

// ---------------------------------------------------------------------------
// adding up
// ---------------------------------------------------------------------------
constexpr int LONGEST_RUN = 32, SHORTEST_RUN = 8;      // sorted positions per wave

struct SumArgs {
    void* dW;
    const void* err;
    const uint2* sorted;
    const uint32_t* present;
    uint32_t* total;             // positions; entries of the two lists
    uint4* joins;                // words to join: (first run, last run, word); few runs, then, from the end, many
    uint32_t runs;
    float* part;                 // [run][head, tail][embed]
    float scale, beta;
    uint32_t embed, vocab, words_per, tiles;
    uint32_t count, list_blocks, sum_blocks;
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

// A wave clears (or scales) the absent ones of 16 consecutive words.
constexpr int CLEAR_ROWS = 16;
template <typename T> NEON_DEV void clear_rows(const SumArgs& a, uint32_t block) {
    constexpr int V = vec<T>::V;
    const int lane = threadIdx.x & 63;
    const size_t w0 = ((size_t)block * 4 + (threadIdx.x >> 6)) * CLEAR_ROWS;
    bool absent = false;
    if (lane < CLEAR_ROWS && w0 + lane < a.vocab) {
        const uint32_t w = (uint32_t)(w0 + lane), local = w >> CLASS_LOG;
        absent = !((a.present[(size_t)(w & (CLASSES - 1)) * a.words_per + (local >> 5)] >> (local & 31)) & 1u);
    }
    const float zero[V] = {};
    for (unsigned long long todo = __ballot(absent); todo; todo &= todo - 1) {
        T* row = (T*)a.dW + (w0 + __builtin_ctzll(todo)) * a.ld_dw;
        for (uint32_t c = lane * V; c < a.embed; c += 64 * V)
            put_row<T, V>(row + c, zero, a.embed - c >= V ? V : (int)(a.embed - c), 0.0f, a.beta);
    }
}

// A thread per run: does a word begin in it and go on behind it?  Then its last
// run (run k begins at k * RUN; the runs that begin with the word follow one
// another, so their end is found in a few rounds of probes, the probes of a round
// in flight together), and an entry in the
// list of the waves or of the workgroups of lut_join_kernel.  The order of the
// lists is any, what becomes of their entries is not.
constexpr uint32_t MANY_RUNS = 24;        // (three rounds of eight loads for a wave)
template <int RUN> NEON_DEV void list_words(const SumArgs& a, uint32_t total) {
    const size_t run = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t s0 = run * RUN;
    if (s0 + RUN >= total) return;
    const uint32_t word = a.sorted[s0 + RUN].x;
    if (a.sorted[s0 + RUN - 1].x != word || (s0 > 0 && a.sorted[s0 - 1].x == word)) return;
    const uint32_t borders = (total + RUN - 1) / RUN;
    const auto goes_on = [&](unsigned long long k) { return k < borders && a.sorted[k * RUN].x == word; };
    unsigned long long in = run + 1, out = borders;          // the last run lies in [in, out)
    bool hit[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) hit[i] = goes_on(run + 1 + (1u << i));
#pragma unroll
    for (int i = 15; i >= 0; --i) {
        if (!hit[i] && run + 1 + (1u << i) < out) out = run + 1 + (1u << i);
        if (hit[i] && run + 1 + (1u << i) > in) in = run + 1 + (1u << i);
    }
    while (out - in > 1) {
        const unsigned long long step = (out - in + 7) / 8, from = in;
#pragma unroll
        for (int i = 0; i < 7; ++i) hit[i] = from + (i + 1) * step < out && goes_on(from + (i + 1) * step);
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            const unsigned long long k = from + (i + 1) * step;
            if (hit[i]) in = k;
            else if (k < out) out = k;
        }
    }
    const bool many = in - run > MANY_RUNS;
    const uint32_t at = atomicAdd(a.total + (many ? 2 : 1), 1u);
    a.joins[many ? a.runs - 1 - at : at] = make_uint4((uint32_t)run, (uint32_t)in, word, 0);
}

// Workgroups: list_blocks that look for words to join, sum_blocks that add, and
// the rest clears.
template <typename T, int RUN> __global__ __launch_bounds__(256) void lut_sum_kernel(SumArgs a) {
    constexpr int V = vec<T>::V;
    if (blockIdx.x >= a.list_blocks + a.sum_blocks) {
        clear_rows<T>(a, blockIdx.x - a.list_blocks - a.sum_blocks);
        return;
    }
    if (blockIdx.x < a.list_blocks) {
        list_words<RUN>(a, a.total[0]);
        return;
    }
    const int lane = threadIdx.x & 63;
    const uint32_t id = (blockIdx.x - a.list_blocks) * 4 + (threadIdx.x >> 6);
    const uint32_t run = id / a.tiles;
    if (run >= a.runs) return;
    const uint32_t c = (id % a.tiles * 64 + lane) * V;
    const size_t s0 = (size_t)run * RUN;
    // lane i: entry i; lane 62: the entry before the run, lane 63: the one after it (the entries behind the
    // total hold anything; they are there, and taken for no word)
    const long long mine = lane < RUN ? (long long)s0 + lane : lane == 62 ? (long long)s0 - 1 : lane == 63 ? (long long)s0 + RUN : -1;
    uint2 item = make_uint2(NO_WORD, 0);
    if (mine >= 0 && mine < (long long)a.count) item = a.sorted[mine];
    const uint32_t total = a.total[0];
    if (s0 >= total) return;
    if (mine >= (long long)total) item = make_uint2(NO_WORD, 0);
    const int len = total - s0 < RUN ? (int)(total - s0) : RUN;
    const int n = c >= a.embed ? 0 : (a.embed - c >= V ? V : (int)(a.embed - c));
    const T* err = (const T*)a.err + c;
    // bit i: entry i is the last of its word in this run
    const uint32_t next = (uint32_t)__shfl((int)item.x, lane == RUN - 1 ? 63 : lane + 1);
    const unsigned long long ends = __ballot(lane < len && (next != item.x || lane == len - 1));
    bool head = __builtin_amdgcn_readlane((int)item.x, 0) == __builtin_amdgcn_readlane((int)item.x, 62);   // began before
    const bool on = len == RUN && __builtin_amdgcn_readlane((int)item.x, RUN - 1) == __builtin_amdgcn_readlane((int)item.x, 63);
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    constexpr int AHEAD = 8;          // (16: 37.6 us instead of 36.3 for 32768 x 1024 bf16)
    for (int i0 = 0; i0 < len; i0 += AHEAD) {
        nh_raw<T, V> r[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int e = i0 + i < len ? i0 + i : len - 1;
            const T* row = err + (size_t)(uint32_t)__builtin_amdgcn_readlane((int)item.y, e) * a.ld_err;
            if (n == V) r[i].load(row);
            else if (n > 0) r[i].load_partial(row, n);
            else r[i].zero();
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (i0 + i >= len) break;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += r[i].get(k);
            if (!((ends >> (i0 + i)) & 1ull)) continue;
            const bool goes_on = on && i0 + i == RUN - 1;
            if (n > 0) {
                if (head || goes_on) {
                    float* p = a.part + ((size_t)run * 2 + (head ? 0 : 1)) * a.embed + c;
                    if (n == V) {
                        nh_store_vec<float, V>(p, acc);
                    } else {
#pragma unroll
                        for (int k = 0; k < V; ++k)
                            if (k < n) p[k] = acc[k];
                    }
                } else {
                    const uint32_t word = (uint32_t)__builtin_amdgcn_readlane((int)item.x, i0 + i);
                    put_row<T, V>((T*)a.dW + (size_t)word * a.ld_dw + c, acc, n, a.scale, a.beta);
                }
            }
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = 0.0f;
            head = false;
        }
    }
}

// The words that go on behind the run they begin in: tail of that run + heads
// of the following ones, 256 columns at a time.  A word of few runs is one
// wave's; the runs of the others are dealt to the waves of a workgroup in
// contiguous shares, and the shares joined in order.
constexpr int JOIN_T = 1024, JOIN_W = JOIN_T / 64;
constexpr unsigned JOIN_BLOCKS = 128;       // per 256 columns

NEON_DEV void add_part(const float* p, int n, float (&acc)[4]) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n == 4) nh_load_vec<float, 4>(p, v);
    else
        for (int k = 0; k < n; ++k) v[k] = p[k];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] += v[k];
}
NEON_DEV void add_tail(const SumArgs& a, size_t run, uint32_t c, int n, float (&acc)[4]) {
    add_part(a.part + (run * 2 + 1) * a.embed + c, n, acc);
}
NEON_DEV void add_heads(const SumArgs& a, size_t h0, size_t h1, uint32_t c, int n, float (&acc)[4]) {
#pragma unroll 8
    for (size_t h = h0; h < h1; ++h) add_part(a.part + h * 2 * a.embed + c, n, acc);
}

template <typename T> __global__ __launch_bounds__(JOIN_T) void lut_join_kernel(SumArgs a) {
    __shared__ float share[JOIN_W][256];
    const uint32_t few = a.total[1], many = a.total[2];
    const uint32_t tiles = (a.embed + 255) / 256, block = blockIdx.x / tiles, blocks = gridDim.x / tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t c = (blockIdx.x % tiles) * 256 + lane * 4;
    const int n = c >= a.embed ? 0 : (a.embed - c >= 4 ? 4 : (int)(a.embed - c));
    for (uint32_t item = block; item < many; item += blocks) {
        const uint4 it = a.joins[a.runs - 1 - item];
        const size_t per = (it.y - it.x + JOIN_W - 1) / JOIN_W;
        const size_t h0 = it.x + 1 + (size_t)wave * per, h1 = h0 + per < (size_t)it.y + 1 ? h0 + per : (size_t)it.y + 1;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (wave == 0) add_tail(a, it.x, c, n, acc);
        add_heads(a, h0, h1, c, n, acc);
#pragma unroll
        for (int k = 0; k < 4; ++k) share[wave][lane * 4 + k] = acc[k];
        __syncthreads();
        if (wave == 0 && n > 0) {
#pragma unroll
            for (int w = 1; w < JOIN_W; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] += share[w][lane * 4 + k];
            put_row<T, 4>((T*)a.dW + (size_t)it.z * a.ld_dw + c, acc, n, a.scale, a.beta);
        }
        __syncthreads();
    }
    if (n == 0) return;
    for (uint32_t item = block + blocks * wave; item < few; item += blocks * JOIN_W) {
        const uint4 it = a.joins[item];
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        add_tail(a, it.x, c, n, acc);
        add_heads(a, (size_t)it.x + 1, (size_t)it.y + 1, c, n, acc);
        put_row<T, 4>((T*)a.dW + (size_t)it.z * a.ld_dw + c, acc, n, a.scale, a.beta);
    }
}

// ---------------------------------------------------------------------------
// workspace of the gradient
// ---------------------------------------------------------------------------
struct Layout {
    size_t split, table, scratch, sorted, present, total, joins, part, turned, bytes;
    uint32_t words_per;
    int run;              // sorted positions per wave of lut_sum_kernel
};

// Waves of lut_sum_kernel below which it takes shorter runs: eight per CU.  Sums + joining in us, in runs of 32,
// 16 and 8: 32768 x 1024 bf16 (2048 waves of 32) 36 + 6, 39 + 7; 8192 x 4096 bf16 (2048) 72 + 7, 72 + 8; 16384
// x 300 fp32 (1024) 20 + 5, 15 + 6, 17 + 7; 65536 x 128 fp32 (2048) 34 + 6, 30 + 7.
constexpr size_t SUM_WAVES = 2048;

Layout layout(int dtype, int axis, size_t count, size_t embed, size_t vocab) {
    Layout l;
    size_t at = 0;
    const auto take = [&at](size_t bytes) {
        const size_t here = at;
        at += lm::align256(bytes);
        return here;
    };
    l.words_per = (uint32_t)lm::ceil_div(lm::ceil_div(vocab, CLASSES), 32);
    l.split = take(count * sizeof(uint2));
    l.table = take(lm::ceil_div(count, SLICE) * (CLASSES + 1) * 4);
    l.scratch = take(count * sizeof(uint2));
    l.sorted = take(count * sizeof(uint2));
    l.present = take((size_t)CLASSES * l.words_per * 4);
    l.total = take(12);
    l.run = LONGEST_RUN;
    while (l.run > SHORTEST_RUN && lm::ceil_div(count, l.run) * lm::ceil_div(embed, 64 * (16 / lm::item_bytes(dtype))) < SUM_WAVES)
        l.run /= 2;
    l.joins = take(lm::ceil_div(count, l.run) * sizeof(uint4));
    l.part = take(lm::ceil_div(count, l.run) * 2 * embed * sizeof(float));
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
    const uint32_t pad = pad_word(pad_idx), words = (uint32_t)vocab, cols = (uint32_t)embed;
    return lm::run(who, stream, [&](lm::Launches& launch) {
        lm::by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr size_t V = vec<T>::V;
            if (axis == 1) {
                int log = 0;
                while (log < 8 && ((size_t)V << log) < embed) ++log;
                launch(lut_rows_fprop_kernel<T>, lm::ceil_div(positions, (size_t)256 >> log), 1, 256, 0, (T*)out, (const T*)W, ids,
                       scale, positions, cols, words, pad, ld_w, ld_out, log);
            } else {
                launch(lut_cols_fprop_kernel<T>, lm::ceil_div(positions, TURN_POS) * lm::ceil_div(embed, 8 * V), 1, 256, 0, (T*)out,
                       (const T*)W, ids, scale, positions, cols, words, pad, ld_w, ld_out);
            }
        });
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
    if (!lm::aligned16(workspace)) return lm::refuse(who, "workspace off a 16-byte boundary");
    char* ws = (char*)workspace;
    return lm::run(who, stream, [&](lm::Launches& launch) {
        lm::by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr size_t V = vec<T>::V;
            SortArgs q = {};
            q.ids = ids;
            q.split = (uint2*)(ws + l.split);
            q.table = (uint32_t*)(ws + l.table);
            q.scratch = (uint2*)(ws + l.scratch);
            q.sorted = (uint2*)(ws + l.sorted);
            q.present = (uint32_t*)(ws + l.present);
            q.total = (uint32_t*)(ws + l.total);
            q.count = (uint32_t)positions;
            q.slices = (uint32_t)lm::ceil_div(positions, SLICE);
            q.vocab = (uint32_t)vocab;
            q.pad = pad_word(pad_idx);
            q.words_per = l.words_per;
            for (size_t rest = (vocab - 1) >> CLASS_LOG; rest; rest >>= 8) ++q.passes;
            SumArgs a = {};
            a.dW = dW;
            a.err = err;
            a.ld_err = ld_err;
            TurnArgs turned = {};
            size_t turning = 0;
            if (axis == 0) {
                turned.from = err;
                turned.to = ws + l.turned;
                turned.count = (uint32_t)positions;
                turned.embed = (uint32_t)embed;
                turned.tiles_e = (uint32_t)lm::ceil_div(embed, turn<T>::E);
                turned.ld = ld_err;
                turning = turned.tiles_e * lm::ceil_div(positions, turn<T>::P);
                a.err = ws + l.turned;
                a.ld_err = embed;
            }
            if (positions) launch(lut_split_kernel<T>, q.slices + turning, 1, SORT_T, 0, q, turned);
            launch(lut_class_kernel, CLASSES, 1, SORT_T, 0, q);
            a.sorted = q.sorted;
            a.present = q.present;
            a.total = q.total;
            a.joins = (uint4*)(ws + l.joins);
            a.part = (float*)(ws + l.part);
            a.scale = scale;
            a.beta = beta;
            a.embed = (uint32_t)embed;
            a.vocab = (uint32_t)vocab;
            a.words_per = l.words_per;
            a.ld_dw = ld_dw;
            a.tiles = (uint32_t)lm::ceil_div(embed, 64 * V);
            const size_t runs = lm::ceil_div(positions, l.run);
            a.runs = (uint32_t)runs;
            const size_t adding = lm::ceil_div(runs * a.tiles, 4), joining = (runs < JOIN_BLOCKS ? runs : JOIN_BLOCKS) * lm::ceil_div(embed, 256);
            const size_t clearing = beta == 1.0f ? 0 : lm::ceil_div(vocab, 4 * CLEAR_ROWS);
            const size_t listing = runs > 1 ? lm::ceil_div(runs, 256) : 0;
            a.count = (uint32_t)positions;
            a.list_blocks = (uint32_t)listing;
            a.sum_blocks = (uint32_t)adding;
            const auto go = [&](auto run) {
                constexpr int RUN = decltype(run)::value;
                if (adding + clearing) launch(lut_sum_kernel<T, RUN>, listing + adding + clearing, 1, 256, 0, a);
                if (runs > 1) launch(lut_join_kernel<T>, joining, 1, JOIN_T, 0, a);
            };
            if (l.run == 32) go(std::integral_constant<int, 32>());
            else if (l.run == 16) go(std::integral_constant<int, 16>());
            else go(std::integral_constant<int, 8>());
        });
    });
}

}  // extern "C"
