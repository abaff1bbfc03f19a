// Distillation from a teacher's top logits.  Position n has a student's logits
// z over the whole vocabulary and K teacher entries (word id, logit t); entries
// whose id lies outside the vocabulary do not count.  With a temperature T
//
//   p = softmax over the entries of t / T        q = softmax over the vocabulary of z / T
//   loss = T^2 sum_k p_k (log p_k - log q[id_k])
//   dz_v = w T (q_v - sum of p_k over the entries with id_k == v)
//
// A position without entries (or whose t are all -inf) has loss 0 and gradient
// 0, whatever its logits hold.  Forward reads z once and also leaves what
// backward starts from: the largest z and the logarithm of the sum of
// exp((z - largest) / T), and the same of the entries.  (Two numbers each, not
// their sum: in a log-sum-exp of logits around 1e6 fp32 has no digits left for
// the logarithm.)  Backward reads z once and writes dz once.  HBM traffic bounds
// both.
//
// Layouts: "rows" (a position's logits lie side by side) and "columns"
// (positions lie side by side, the backend's usual layout).
#include "lm_ops.h"

namespace {

using lm::vec;

constexpr int MOST_ENTRIES = NH_DISTILL_MAX_ENTRIES;
constexpr float LOG2E = 1.44269502f;

struct DistillArgs {
    const void* z;
    void* dz;
    const int32_t* ids;
    const void* t;
    float* loss;
    float* stats;           // four vectors: largest z, log sum, largest t (-inf without entries), log sum
    long long stat_k;       // from one of them to the next
    const float* weight;    // nullptr: weight_all
    float weight_all;
    float inv_t, temperature;
    int t_dtype;
    uint32_t vocab, entries;
    size_t positions, ld_z, ld_dz;
    long long ids_k, ids_n, t_k, t_n;           // strides of the entry tensors
    long long loss_n, stat_n, weight_n;
    nh_pair* part;          // forward: (maximum, sum) per position and chunk
    uint32_t chunk, chunks;
};

NEON_DEV float load_t(const DistillArgs& a, uint32_t k, size_t n) {
    const long long at = (long long)k * a.t_k + (long long)n * a.t_n;
    if (a.t_dtype == NH_T_F32) return ((const float*)a.t)[at];
    if (a.t_dtype == NH_T_F16) return (float)((const nh_f16*)a.t)[at];
    return (float)((const nh_bf16*)a.t)[at];
}
NEON_DEV int load_id(const DistillArgs& a, uint32_t k, size_t n) {
    return a.ids[(long long)k * a.ids_k + (long long)n * a.ids_n];
}
struct Stats {
    float top, log_sum, t_top, t_log_sum;
};
NEON_DEV Stats load_stats(const DistillArgs& a, size_t n) {
    const float* p = a.stats + (long long)n * a.stat_n;
    return {p[0], p[a.stat_k], p[2 * a.stat_k], p[3 * a.stat_k]};
}
NEON_DEV float entry_p(const DistillArgs& a, float t, const Stats& s) { return expf((t - s.t_top) * a.inv_t - s.t_log_sum); }
NEON_DEV bool is_word(int id, uint32_t vocab) { return (uint32_t)id < vocab; }

// (m, s): largest logit seen and sum of e^((z - m) / T).  A state that has seen nothing but
// -inf keeps s = 0; NaN and +inf make s NaN, as in the two-sweep form.
struct Lse {
    float m, s;
};
NEON_DEV Lse lse_join(Lse a, Lse b, float c) {
    Lse r;
    r.m = nh_max(a.m, b.m);
    const float z = r.m == -NH_INF ? 0.0f : r.m;
    r.s = a.s * __builtin_amdgcn_exp2f((a.m - z) * c) + b.s * __builtin_amdgcn_exp2f((b.m - z) * c);
    return r;
}
template <int N> NEON_DEV void lse_add(Lse& a, const float (&x)[N], float c) {
    float m = a.m;
#pragma unroll
    for (int i = 0; i < N; ++i) m = nh_max(m, x[i]);
    const float z = m == -NH_INF ? 0.0f : m;
    float s = a.s * __builtin_amdgcn_exp2f((a.m - z) * c);
#pragma unroll
    for (int i = 0; i < N; ++i) s += __builtin_amdgcn_exp2f((x[i] - z) * c);
    a.m = m;
    a.s = s;
}
// over the 64 lanes; every lane gets the same bits (the two partners join in lane order)
NEON_DEV Lse lse_wave(Lse v, float c) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        Lse o;
        o.m = __shfl_xor(v.m, d);
        o.s = __shfl_xor(v.s, d);
        v = (threadIdx.x & d) ? lse_join(o, v, c) : lse_join(v, o, c);
    }
    return v;
}
NEON_DEV float wave_sum(float v) { return nh_wave_allreduce<nh_op_sum, 64>(v); }
NEON_DEV float wave_max(float v) { return nh_wave_allreduce<nh_op_max, 64>(v); }

// where a position's entries are read from
struct InMemory {
    const DistillArgs& a;
    size_t n;
    NEON_DEV int id(uint32_t k) const { return load_id(a, k, n); }
    NEON_DEV float t(uint32_t k) const { return load_t(a, k, n); }
};
struct InLds {
    const int* ids;
    const float* ts;
    NEON_DEV int id(uint32_t k) const { return ids[k]; }
    NEON_DEV float t(uint32_t k) const { return ts[k]; }
};

// One wave, with the student's state of position n: the teacher's entries, the
// loss and the statistics.  z[v * step] is the logit of word v.
template <typename T, class E>
NEON_DEV void finish_position(const DistillArgs& a, size_t n, Lse st, const T* z, size_t step, const E& entry) {
    const int lane = threadIdx.x & 63;
    const float log_s = logf(st.s);
    float top = -NH_INF;
    for (uint32_t k = lane; k < a.entries; k += 64)
        if (is_word(entry.id(k), a.vocab)) top = nh_max(top, entry.t(k));
    top = wave_max(top);
    const bool some = top != -NH_INF;
    const float top0 = some ? top : 0.0f;
    float sum = 0.0f;
    for (uint32_t k = lane; k < a.entries; k += 64)
        if (is_word(entry.id(k), a.vocab)) sum += expf((entry.t(k) - top0) * a.inv_t);
    sum = wave_sum(sum);
    const float log_t = logf(sum);
    float loss = 0.0f;
    for (uint32_t k = lane; k < a.entries && some; k += 64) {
        const int id = entry.id(k);
        if (!is_word(id, a.vocab)) continue;
        const float log_p = (entry.t(k) - top0) * a.inv_t - log_t;
        const float p = expf(log_p);
        const float log_q = ((float)z[(size_t)id * step] - st.m) * a.inv_t - log_s;
        if (p != 0.0f) loss = __builtin_fmaf(p, log_p - log_q, loss);
    }
    loss = wave_sum(loss);
    if (lane == 0) {
        a.loss[(long long)n * a.loss_n] = a.temperature * a.temperature * loss;
        float* p = a.stats + (long long)n * a.stat_n;
        p[0] = st.m;
        p[a.stat_k] = log_s;
        p[2 * a.stat_k] = top;
        p[3 * a.stat_k] = log_t;
    }
}

// PAST: the logits are more than the last-level cache holds, read and written past it.  (A parameter of
// the kernels: of two branches that differ in that alone the compiler makes one, without it.)
template <bool PAST, typename T, int V> NEON_DEV void load_logits(nh_raw<T, V>& r, const T* p) {
    if constexpr (PAST) r.load_stream(p);
    else r.load(p);
}
template <bool PAST, typename T, int V> NEON_DEV void store_grads(const nh_out<T, V>& o, T* p) {
    if constexpr (PAST) o.store_stream(p);
    else o.store(p);
}

// ---------------------------------------------------------------------------
// forward: (maximum, sum) of chunks of the vocabulary.  A position whose
// vocabulary is one chunk is finished by the same workgroup; otherwise one wave
// per position joins the chunks in order.  4096 x 50001 bf16, 410 MB: 87 us (4.7
// TB/s), about half of that time in the exponentials; 4096 x 32000 fp32, 524 MB: 87
// us (6.0 TB/s).  In chunks of 16 KB the former took a seventh more, the fold over
// the lanes being paid for each.
// ---------------------------------------------------------------------------
template <typename T, bool PAST> __global__ __launch_bounds__(256) void distill_rows_lse_kernel(DistillArgs a) {
    constexpr int V = vec<T>::V, AHEAD = 4;
    __shared__ Lse slots[4];
    const size_t n = blockIdx.x / a.chunks;
    const uint32_t i0 = (blockIdx.x % a.chunks) * a.chunk;
    const uint32_t i1 = i0 + a.chunk < a.vocab ? i0 + a.chunk : a.vocab;
    const T* z = (const T*)a.z + n * a.ld_z;
    const float c = a.inv_t * LOG2E;
    Lse st = {-NH_INF, 0.0f};
    // batches of AHEAD vectors per thread, the next one on its way while one is added up
    constexpr uint32_t BATCH = AHEAD * 256 * V;
    const uint32_t batches = (i1 - i0) / BATCH;
    uint32_t i = i0 + threadIdx.x * V;
    nh_raw<T, V> even[AHEAD], odd[AHEAD];
    const auto load = [&](nh_raw<T, V> (&r)[AHEAD], uint32_t at) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) load_logits<PAST>(r[k], z + at + k * 256 * V);
    };
    const auto add = [&](const nh_raw<T, V> (&r)[AHEAD]) {
        float x[AHEAD * V];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) x[k * V + j] = r[k].get(j);
        lse_add<AHEAD * V>(st, x, c);
    };
    if (batches) load(even, i);
    for (uint32_t b = 0; b < batches; b += 2) {
        if (b + 1 < batches) load(odd, i + BATCH);
        add(even);
        if (b + 1 < batches) {
            if (b + 2 < batches) load(even, i + 2 * BATCH);
            add(odd);
        }
        i += 2 * BATCH;
    }
    i = i0 + batches * BATCH + threadIdx.x * V;
    for (; i < i1; i += 256 * V) {
        nh_raw<T, V> r;
        const int left = i1 - i < V ? (int)(i1 - i) : V;
        if (left == V) r.load(z + i);
        else r.load_partial(z + i, left);
        float x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = j < left ? r.get(j) : -NH_INF;
        lse_add<V>(st, x, c);
    }
    st = lse_wave(st, c);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = st;
    __syncthreads();
    if (threadIdx.x < 64) {
        st = lse_join(lse_join(slots[0], slots[1], c), lse_join(slots[2], slots[3], c), c);
        if (a.chunks == 1) {
            finish_position(a, n, st, z, 1, InMemory{a, n});
            return;
        }
        nh_pair p;
        p.v = st.m;
        p.i = __builtin_bit_cast(int, st.s);
        if (threadIdx.x == 0) a.part[(size_t)blockIdx.x] = p;      // [n][chunk]
    }
}

constexpr int LC = 8;       // lanes across a strip of 128 bytes of positions
template <typename T> struct strip { static constexpr int COLS = LC * vec<T>::V; };

template <typename T> __global__ __launch_bounds__(256) void distill_cols_lse_kernel(DistillArgs a) {
    constexpr int V = vec<T>::V, COLS = strip<T>::COLS, RL = 256 / LC, AHEAD = 8;
    __shared__ Lse slots[4][COLS];
    const uint32_t strips = gridDim.x / a.chunks;        // (neighbouring workgroups: neighbouring memory)
    const size_t c0 = (size_t)(blockIdx.x % strips) * COLS;
    const uint32_t chunk = blockIdx.x / strips;
    const uint32_t i0 = chunk * a.chunk, i1 = i0 + a.chunk < a.vocab ? i0 + a.chunk : a.vocab;
    const int cl = threadIdx.x % LC, rl = threadIdx.x / LC;
    const size_t col = c0 + cl * V;
    const int n = col >= a.positions ? 0 : (a.positions - col >= V ? V : (int)(a.positions - col));
    const T* z = (const T*)a.z + col;
    const float c = a.inv_t * LOG2E;
    Lse st[V];
#pragma unroll
    for (int j = 0; j < V; ++j) st[j] = {-NH_INF, 0.0f};
    if (n > 0)
        for (uint32_t i = i0 + rl; i < i1; i += AHEAD * RL) {
            nh_raw<T, V> r[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const uint32_t f = i + k * RL;
                if (f >= i1) r[k].zero();
                else if (n == V) r[k].load(z + (size_t)f * a.ld_z);
                else r[k].load_partial(z + (size_t)f * a.ld_z, n);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float x[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) x[k] = i + k * RL < i1 ? r[k].get(j) : -NH_INF;
                lse_add<AHEAD>(st[j], x, c);
            }
        }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int d = LC; d < 64; d <<= 1) {
            Lse o;
            o.m = __shfl_xor(st[j].m, d);
            o.s = __shfl_xor(st[j].s, d);
            st[j] = (threadIdx.x & d) ? lse_join(o, st[j], c) : lse_join(st[j], o, c);
        }
        if ((threadIdx.x & 63) < LC) slots[threadIdx.x >> 6][cl * V + j] = st[j];
    }
    __syncthreads();
    if (threadIdx.x < COLS && c0 + threadIdx.x < a.positions) {
        const int x = threadIdx.x;
        const Lse r = lse_join(lse_join(slots[0][x], slots[1][x], c), lse_join(slots[2][x], slots[3][x], c), c);
        nh_pair p;
        p.v = r.m;
        p.i = __builtin_bit_cast(int, r.s);
        a.part[(c0 + x) * a.chunks + chunk] = p;
    }
}

// Positions whose vocabulary was split, and the columns layout: `group` positions
// per workgroup (a multiple of its four waves), their entries brought to LDS side
// by side -- in the columns layout an entry's neighbours in memory are other
// positions', and 16 of them share a cache line.
template <typename T> __global__ __launch_bounds__(256) void distill_finish_kernel(DistillArgs a, size_t z_n, size_t z_v, bool rows,
                                                                                  uint32_t group) {
    extern __shared__ int entries[];          // ids, then t: [position][entry]
    float* ts = (float*)(entries + group * a.entries);
    const size_t n0 = (size_t)blockIdx.x * group;
    const uint32_t all = group * a.entries;
    for (uint32_t i = threadIdx.x; i < all; i += 256) {
        const uint32_t x = rows ? i / a.entries : i % group, k = rows ? i % a.entries : i / group;
        if (n0 + x >= a.positions) continue;
        entries[x * a.entries + k] = load_id(a, k, n0 + x);
        ts[x * a.entries + k] = load_t(a, k, n0 + x);
    }
    __syncthreads();
    const float c = a.inv_t * LOG2E;
    for (uint32_t x = threadIdx.x >> 6; x < group; x += 4) {
        const size_t n = n0 + x;
        if (n >= a.positions) return;
        Lse st = {-NH_INF, 0.0f};
        for (uint32_t i = threadIdx.x & 63; i < a.chunks; i += 64) {
            const nh_pair p = a.part[n * a.chunks + i];
            st = lse_join(st, {p.v, __builtin_bit_cast(float, p.i)}, c);
        }
        finish_position(a, n, lse_wave(st, c), (const T*)a.z + n * z_n, z_v,
                        InLds{entries + x * a.entries, ts + x * a.entries});
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
NEON_DEV float weight_of(const DistillArgs& a, size_t n) {
    return (a.weight ? a.weight[(long long)n * a.weight_n] : a.weight_all) * a.temperature;
}
NEON_DEV float prob_q(float z, float inv_t, float top, float log_sum) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(z - top, inv_t, -log_sum) * LOG2E);
}

// Which of a position's words are named more than once: a table of word ids in
// LDS with at least twice as many places as entries, open addressing.  Returns
// the place of `id`; `twice` gets a bit for a place that was asked for again.
NEON_DEV uint32_t table_size(uint32_t entries) {
    uint32_t n = 64;
    while (n < 2 * entries) n *= 2;
    return n;
}
NEON_DEV uint32_t table_put(int* table, uint32_t* twice, uint32_t size, int id) {
    uint32_t at = ((uint32_t)id * 2654435761u >> 16) & (size - 1);
    for (;;) {
        const int old = atomicCAS(&table[at], -1, id);
        if (old == -1) return at;
        if (old == id) {
            atomicOr(&twice[at >> 5], 1u << (at & 31));
            return at;
        }
        at = (at + 1) & (size - 1);
    }
}
// (is entry k the first with its word?, the sum over all of them), for words named more than once
NEON_DEV bool first_and_sum(const int* ids, const float* ps, uint32_t entries, uint32_t k, float& p) {
    const int id = ids[k];
    bool first = true;
    p = 0.0f;
    for (uint32_t o = 0; o < entries; ++o)
        if (ids[o] == id) {
            first = first && o >= k;
            p += ps[o];
        }
    return first;
}
constexpr int MOST_PLACES = 2 * MOST_ENTRIES;

// One workgroup per position and chunk of the vocabulary (four 16-byte vectors
// per thread at most, all asked for before anything else): w T q over the chunk,
// then the few words of the chunk that the teacher names once more with p in.
// Bound by HBM: 8192 x 32000 bf16, 1.05 GB: 178 to 183 us (5.7 to 5.9 TB/s).
constexpr size_t ROW_CHUNK_BYTES = 16384;
template <typename T, bool PAST> __global__ __launch_bounds__(256) void distill_rows_bprop_kernel(DistillArgs a) {
    constexpr int V = vec<T>::V, VECS = ROW_CHUNK_BYTES / 16 / 256;
    __shared__ int ids[MOST_ENTRIES], table[MOST_PLACES];
    __shared__ float ps[MOST_ENTRIES];
    __shared__ uint32_t twice[MOST_PLACES / 32];
    const size_t n = blockIdx.x / a.chunks;
    const uint32_t i0 = (blockIdx.x % a.chunks) * a.chunk;
    const uint32_t i1 = i0 + a.chunk < a.vocab ? i0 + a.chunk : a.vocab;
    const T* z = (const T*)a.z + n * a.ld_z;
    T* dz = (T*)a.dz + n * a.ld_dz;
    // vector k of this thread, of `whole` in the chunk
    const uint32_t whole = (i1 - i0) / V, rest = (i1 - i0) % V;
    const auto at = [&](int k) { return k * 256 + threadIdx.x; };
    nh_raw<T, V> r[VECS];
#pragma unroll
    for (int k = 0; k < VECS; ++k)
        if (at(k) < whole) load_logits<PAST>(r[k], z + i0 + at(k) * V);
    const Stats st = load_stats(a, n);
    const bool some = st.t_top != -NH_INF;
    const float w = weight_of(a, n);
    const uint32_t places = table_size(a.entries);
    for (uint32_t k = threadIdx.x; k < a.entries && some; k += 256) {
        ids[k] = load_id(a, k, n);
        ps[k] = entry_p(a, load_t(a, k, n), st);
    }
    for (uint32_t k = threadIdx.x; k < places; k += 256) table[k] = -1;
    if (threadIdx.x < places / 32) twice[threadIdx.x] = 0;
    const auto grad = [&](float x) { return some ? w * prob_q(x, a.inv_t, st.top, st.log_sum) : 0.0f; };
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
        if (at(k) >= whole) break;
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int j = 0; j < V; ++j) o.set(j, grad(r[k].get(j)));
        store_grads<PAST>(o, dz + i0 + at(k) * V);
    }
    if (threadIdx.x < rest) {        // what is left of a vector, a word each
        const uint32_t i = i0 + whole * V + threadIdx.x;
        dz[i] = nh_store_cvt<T>::f(grad((float)z[i]));
    }
    if (!some) return;
    __syncthreads();        // the entries are in LDS, and the chunk is written before its words are written again
    constexpr int EACH = MOST_ENTRIES / 256;
    uint32_t place[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const uint32_t k = threadIdx.x + 256 * e;
        place[e] = ~0u;
        if (k < a.entries && (uint32_t)ids[k] >= i0 && (uint32_t)ids[k] < i1) place[e] = table_put(table, twice, places, ids[k]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        if (place[e] == ~0u) continue;
        const uint32_t k = threadIdx.x + 256 * e, id = (uint32_t)ids[k];
        float p = ps[k];
        if (((twice[place[e] >> 5] >> (place[e] & 31)) & 1u) && !first_and_sum(ids, ps, a.entries, k, p)) continue;
        dz[id] = nh_store_cvt<T>::f(w * (prob_q((float)z[id], a.inv_t, st.top, st.log_sum) - p));
    }
}

// Columns: w T q everywhere, by strips of 256 bytes of positions and chunks of
// the vocabulary; distill_patch_kernel writes the teacher's words once more.
// 20828 x 9950 fp16, 829 MB: 257 us (3.2 TB/s; 1.08 GB moved, lines of 19900 bytes sharing cache lines with
// their neighbours').  Neighbouring workgroups take
// neighbouring strips of the same words; with neighbouring chunks of one strip 346
// us.
constexpr int BLC = 16;
template <typename T> struct bstrip { static constexpr int COLS = BLC * vec<T>::V; };

template <typename T> __global__ __launch_bounds__(256) void distill_cols_bprop_kernel(DistillArgs a) {
    constexpr int V = vec<T>::V, COLS = bstrip<T>::COLS, RL = 256 / BLC, AHEAD = 4;
    const uint32_t strips = gridDim.x / a.chunks;        // (neighbouring workgroups: neighbouring memory)
    const size_t c0 = (size_t)(blockIdx.x % strips) * COLS;
    const uint32_t i0 = blockIdx.x / strips * a.chunk, i1 = i0 + a.chunk < a.vocab ? i0 + a.chunk : a.vocab;
    const size_t col = c0 + threadIdx.x % BLC * V;
    const int n = col >= a.positions ? 0 : (a.positions - col >= V ? V : (int)(a.positions - col));
    if (n == 0) return;
    const T* z = (const T*)a.z + col;
    T* dz = (T*)a.dz + col;
    float top[V], log_sum[V], w[V];
    bool some[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const size_t x = col + (j < n ? j : 0);
        const Stats st = load_stats(a, x);
        top[j] = st.top;
        log_sum[j] = st.log_sum;
        some[j] = st.t_top != -NH_INF;
        w[j] = weight_of(a, x);
    }
    // two sets of registers in turn, as in the rows kernel; words behind the chunk's end are its last one again
    nh_raw<T, V> even[AHEAD], odd[AHEAD];
    const auto load = [&](nh_raw<T, V> (&r)[AHEAD], uint32_t i) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const T* p = z + (size_t)(i + k * RL < i1 ? i + k * RL : i1 - 1) * a.ld_z;
            if (n == V) r[k].load(p);
            else r[k].load_partial(p, n);
        }
    };
    const auto put = [&](const nh_raw<T, V> (&r)[AHEAD], uint32_t i) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const uint32_t f = i + k * RL;
            if (f >= i1) continue;
            nh_out<T, V> o;
            o.clear();
#pragma unroll
            for (int j = 0; j < V; ++j) o.set(j, some[j] ? w[j] * prob_q(r[k].get(j), a.inv_t, top[j], log_sum[j]) : 0.0f);
            T* p = dz + (size_t)f * a.ld_dz;
            if (n < V) o.store_partial(p, n);
            else o.store(p);
        }
    };
    constexpr uint32_t BATCH = AHEAD * RL;
    uint32_t i = i0 + threadIdx.x / BLC;
    if (i < i1) load(even, i);
    while (i < i1) {
        if (i + BATCH < i1) load(odd, i + BATCH);
        put(even, i);
        i += BATCH;
        if (i >= i1) break;
        if (i + BATCH < i1) load(even, i + BATCH);
        put(odd, i);
        i += BATCH;
    }
}

// Columns, after that: the words the teacher names, with p in.  A workgroup
// takes eight positions (in memory an entry's neighbours are other positions');
// a word named twice is its first entry's.
constexpr int PATCH = 8;
size_t patch_lds(size_t entries) {
    size_t places = 64;
    while (places < 2 * entries) places *= 2;
    return PATCH * (entries * 8 + places * 4 + places / 8);
}
template <typename T> __global__ __launch_bounds__(256) void distill_patch_kernel(DistillArgs a) {
    extern __shared__ int lds[];
    const uint32_t places = table_size(a.entries);
    const int x = threadIdx.x % PATCH;
    int* ids = lds + x * a.entries;
    float* ps = (float*)(lds + PATCH * a.entries) + x * a.entries;
    int* table = lds + 2 * PATCH * a.entries + x * places;
    uint32_t* twice = (uint32_t*)(lds + 2 * PATCH * a.entries + PATCH * places) + x * (places / 32);
    const size_t n = (size_t)blockIdx.x * PATCH + x;
    Stats st = {};
    if (n < a.positions) st = load_stats(a, n);
    const bool some = n < a.positions && st.t_top != -NH_INF;
    const uint32_t k0 = threadIdx.x / PATCH;
    constexpr uint32_t STEP = 256 / PATCH;
    for (uint32_t k = k0; k < a.entries; k += STEP) {
        ids[k] = some ? load_id(a, k, n) : -1;
        ps[k] = some ? entry_p(a, load_t(a, k, n), st) : 0.0f;
    }
    for (uint32_t k = k0; k < places; k += STEP) table[k] = -1;
    for (uint32_t k = k0; k < places / 32; k += STEP) twice[k] = 0;
    __syncthreads();
    for (uint32_t k = k0; k < a.entries; k += STEP)
        if (is_word(ids[k], a.vocab)) table_put(table, twice, places, ids[k]);
    __syncthreads();
    if (!some) return;
    const float w = weight_of(a, n);
    for (uint32_t k = k0; k < a.entries; k += STEP) {
        const int id = ids[k];
        if (!is_word(id, a.vocab)) continue;
        float p = ps[k];
        uint32_t at = ((uint32_t)id * 2654435761u >> 16) & (places - 1);
        while (table[at] != id) at = (at + 1) & (places - 1);
        if (((twice[at >> 5] >> (at & 31)) & 1u) && !first_and_sum(ids, ps, a.entries, k, p)) continue;
        const float q = prob_q((float)((const T*)a.z)[(size_t)id * a.ld_z + n], a.inv_t, st.top, st.log_sum);
        ((T*)a.dz)[(size_t)id * a.ld_dz + n] = nh_store_cvt<T>::f(w * (q - p));
    }
}

// ---------------------------------------------------------------------------
// launch geometry: enough workgroups to fill the device, each with enough of
// the vocabulary to pay for its share of the teacher's entries
// ---------------------------------------------------------------------------
// What the last-level cache holds.  Rows of 32000 bf16 logits, backward: 500 positions (64 MB read and
// written) 12.1 us through the caches, 14.7 past them; 1000 positions 26.9 and 26.2; 2500 positions 66.0 and
// 57.4.  Forward: 1500 positions (96 MB) 23.3 and 24.0, 4096 x 50001 90.2 and 86.7.  Columns are always read and written
// through the caches: lines that share a cache line with their neighbours' lose by the other way (20828 x
// 9950 fp16 267 and 303 us).
constexpr size_t STREAM_BYTES = (size_t)256 << 20;

struct Chunks {
    uint32_t len, count;
};
constexpr size_t MAX_CHUNKS = (size_t)1 << 62;        // as many as their least length lets
Chunks split(size_t vocab, size_t lines, size_t wanted, size_t least) {
    size_t n = lm::ceil_div(wanted, lines ? lines : 1);
    const size_t most = lm::ceil_div(vocab, least);
    if (n > most) n = most;
    if (n < 1) n = 1;
    const size_t len = lm::ceil_div(lm::ceil_div(vocab, n), 64) * 64;
    return {(uint32_t)len, (uint32_t)lm::ceil_div(vocab, len)};
}

Chunks fprop_chunks(int dtype, int axis, size_t vocab, size_t positions) {
    // (columns with 1024 or 8192 workgroups, with the finish: 32000 x 8192 bf16 and 32 entries 126 and 132 us, 10000 x
    // 4096 fp32 47.4 and 46.6, 32000 x 256 fp32 15.3 and 15.6)
    if (axis == 1) return split(vocab, positions, 1024, 4096);
    return split(vocab, lm::ceil_div(positions, (size_t)128 / lm::item_bytes(dtype)), 1024, 256);
}
Chunks bprop_chunks(int dtype, int axis, size_t vocab, size_t positions) {
    // rows: what the threads of a workgroup hold at once.  Workgroups that come and go sweep the memory in
    // order; with a row each they stay, and 2048 rows in step with one another take an eighth longer.
    if (axis == 1) return split(vocab, positions, MAX_CHUNKS, ROW_CHUNK_BYTES / lm::item_bytes(dtype));
    // columns: 128 words, two batches (us with 128, 256, 512 words: 20828 x 9950 fp16 267, 273, 296; 32000 x 256 fp32
    // 19.7, 20.1, 23.2; but 32000 x 8192 bf16 297, 250, 249)
    return split(vocab, lm::ceil_div(positions, (size_t)256 / lm::item_bytes(dtype)), MAX_CHUNKS, 128);
}

size_t workspace_bytes(int dtype, int axis, size_t vocab, size_t positions) {
    return positions * fprop_chunks(dtype, axis, vocab, positions).count * sizeof(nh_pair);
}

int check(const char* who, int dtype, int t_dtype, int axis, size_t vocab, size_t positions, size_t entries, float temperature,
          size_t ld_a, size_t ld_b) {
    if (!lm::known_dtype(dtype) || !lm::known_dtype(t_dtype)) return lm::refuse(who, "unknown storage type");
    if (axis != 0 && axis != 1) return lm::refuse(who, "axis is 0 or 1");
    if (vocab == 0 || vocab > 0x7FFFFFFF - 65536) return lm::refuse(who, "between 1 and 2^31 - 65537 words");
    if (positions > (size_t)1 << 40) return lm::refuse(who, "more than 2^40 positions");
    if (entries > MOST_ENTRIES) return lm::refuse(who, "more than NH_DISTILL_MAX_ENTRIES entries per position");
    // (its square multiplies the loss, and its inverse's product with log2(e) the logits: both finite, neither 0)
    if (!(temperature >= 0x1p-60f && temperature <= 0x1p60f))
        return lm::refuse(who, "the temperature lies between 2^-60 and 2^60");
    const size_t len = axis == 1 ? vocab : positions, lines = axis == 1 ? positions : vocab;
    if (lines > 1 && (ld_a < len || ld_b < len)) return lm::refuse(who, "leading dimension shorter than a line");
    return 0;
}

}  // namespace

extern "C" {

size_t nh_distill_workspace_bytes(int dtype, int axis, size_t vocab, size_t positions) {
    const size_t line = axis == 1 ? vocab : positions;
    if (check("nh_distill_workspace_bytes", dtype, dtype, axis, vocab, positions, 0, 1.0f, line, line)) return 0;
    return workspace_bytes(dtype, axis, vocab, positions);
}

int nh_distill_fprop(float* loss, float* stats, const void* z, const int32_t* ids, const void* t,
                     float temperature, int dtype, int t_dtype, int axis, size_t vocab, size_t positions, size_t entries,
                     size_t ld_z, const int64_t* strides, void* workspace, size_t workspace_bytes_given, void* stream) {
    const char* who = "nh_distill_fprop";
    if (int rc = check(who, dtype, t_dtype, axis, vocab, positions, entries, temperature, ld_z, ld_z)) return rc;
    if (positions == 0) return 0;
    if (!loss || !stats || !z || !strides || (entries && (!ids || !t))) return lm::refuse(who, "null pointer");
    const size_t need = workspace_bytes(dtype, axis, vocab, positions);
    if (!workspace || workspace_bytes_given < need) return lm::refuse(who, "workspace smaller than nh_distill_workspace_bytes");
    if (!lm::aligned16(workspace)) return lm::refuse(who, "workspace off a 16-byte boundary");
    const Chunks c = fprop_chunks(dtype, axis, vocab, positions);
    DistillArgs a = {};
    a.z = z; a.ids = ids; a.t = t; a.loss = loss; a.stats = stats;
    a.inv_t = 1.0f / temperature; a.temperature = temperature; a.t_dtype = t_dtype;
    a.vocab = (uint32_t)vocab; a.entries = (uint32_t)entries; a.positions = positions; a.ld_z = ld_z;
    a.ids_k = strides[0]; a.ids_n = strides[1]; a.t_k = strides[2]; a.t_n = strides[3]; a.loss_n = strides[4];
    a.stat_k = strides[5]; a.stat_n = strides[6];
    a.part = (nh_pair*)workspace; a.chunk = c.len; a.chunks = c.count;
    const bool past = vocab * positions * lm::item_bytes(dtype) >= STREAM_BYTES;
    return lm::run(who, stream, [&](lm::Launches& launch) {
        lm::by_dtype(dtype, [&](auto v) {
            using T = decltype(v);
            if (axis == 1) launch(past ? distill_rows_lse_kernel<T, true> : distill_rows_lse_kernel<T, false>, positions * c.count, 1, 256, 0, a);
            else launch(distill_cols_lse_kernel<T>, lm::ceil_div(positions, strip<T>::COLS) * c.count, 1, 256, 0, a);
            if (axis == 1 && c.count == 1) return;
            // (four positions a wave one after another, or one: 256 positions x 32 entries 4.7 us with one, 11 us
            // with four; 8192 x 256 110 us with one, 53 us with four)
            const uint32_t group = positions >= 4096 ? 16 : 4;
            launch(distill_finish_kernel<T>, lm::ceil_div(positions, group), 1, 256, (unsigned)(group * entries * 8), a,
                   axis == 1 ? ld_z : (size_t)1, axis == 1 ? (size_t)1 : ld_z, axis == 1, group);
        });
    });
}

int nh_distill_bprop(void* dz, const void* z, const int32_t* ids, const void* t, const float* stats,
                     const float* weight, float weight_all, float temperature, int dtype, int t_dtype, int axis, size_t vocab,
                     size_t positions, size_t entries, size_t ld_z, size_t ld_dz, const int64_t* strides, void* stream) {
    const char* who = "nh_distill_bprop";
    if (int rc = check(who, dtype, t_dtype, axis, vocab, positions, entries, temperature, ld_z, ld_dz)) return rc;
    if (positions == 0) return 0;
    if (!dz || !stats || !z || !strides || (entries && (!ids || !t))) return lm::refuse(who, "null pointer");
    const Chunks c = bprop_chunks(dtype, axis, vocab, positions);
    DistillArgs a = {};
    a.z = z; a.dz = dz; a.ids = ids; a.t = t; a.stats = const_cast<float*>(stats);
    a.weight = weight; a.weight_all = weight_all;
    a.inv_t = 1.0f / temperature; a.temperature = temperature; a.t_dtype = t_dtype;
    a.vocab = (uint32_t)vocab; a.entries = (uint32_t)entries; a.positions = positions; a.ld_z = ld_z; a.ld_dz = ld_dz;
    a.ids_k = strides[0]; a.ids_n = strides[1]; a.t_k = strides[2]; a.t_n = strides[3]; a.stat_k = strides[4];
    a.stat_n = strides[5]; a.weight_n = strides[6];
    a.chunk = c.len; a.chunks = c.count;
    const bool past = 2 * vocab * positions * lm::item_bytes(dtype) >= STREAM_BYTES;
    return lm::run(who, stream, [&](lm::Launches& launch) {
        lm::by_dtype(dtype, [&](auto v) {
            using T = decltype(v);
            if (axis == 1)
                return launch(past ? distill_rows_bprop_kernel<T, true> : distill_rows_bprop_kernel<T, false>, positions * c.count, 1, 256, 0, a);
            launch(distill_cols_bprop_kernel<T>, lm::ceil_div(positions, bstrip<T>::COLS) * c.count, 1, 256, 0, a);
            if (entries) launch(distill_patch_kernel<T>, lm::ceil_div(positions, PATCH), 1, 256, (unsigned)patch_lds(entries), a);
        });
    });
}

}  // extern "C"
