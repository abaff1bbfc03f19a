// Layer normalisation: statistics of every position over its features.
//
//   forward   mu = mean_f x, var = mean_f (x - mu)^2,  y = gamma (x - mu) r + beta,  r = 1 / sqrt(var + eps)
//   backward  h = (x - mu) r, u = gamma dy
//             dx = r (u - mean_f u - h mean_f(u h)),  dgamma = sum_n dy h,  dbeta = sum_n dy
//
// Two memory layouts: "rows" (features of a position lie side by side) and
// "columns" (positions lie side by side, the backend's usual layout).  Both
// are bound by HBM traffic: forward reads x and writes y, backward reads x and
// dy and writes dx.  Statistics, sums and products are fp32; x, y, dx are
// rounded once, when stored.
#include <type_traits>

#include "lm_ops.h"

namespace {

using lm::vec;

struct LnArgs {
    const void* x;
    const void* dy;       // backward
    void* out;            // y or dx
    const float* gamma;
    const float* beta;    // forward
    float* mean;          // written by forward, read by backward
    float* var;
    float* part;          // workspace
    float* grads[2];      // dgamma, dbeta
    float eps;
    uint32_t features;
    size_t positions;
    size_t ld_x, ld_dy, ld_out;
    bool stream;          // the output is larger than what the caches keep of it
};

// 1 / sqrt(var + eps): the hardware's estimate and one Newton step, within 2
// units in the last place, in place of a square root and a division (thirty
// instructions, of which a thread of the column kernels needs eight in a row).
NEON_DEV float inv_std(float var, float eps) {
    const float v = var + eps;
    float r = __builtin_amdgcn_rsqf(v);
    r = __builtin_fmaf(0.5f * r, __builtin_fmaf(-(v * r), r, 1.0f), r);
    if (__builtin_expect(!(v >= 1.17549435e-38f && v <= NH_FLT_MAX), 0)) {
        asm volatile("");                 // (a branch, not a select)
        r = 1.0f / sqrtf(v);
    }
    return r;
}

// sum over the TPR threads of a row; `slots` (one pair per wave) must not be
// in use by an earlier call whose readers may not have finished
template <int TPR> NEON_DEV void row_sum2(float& a, float& b, float2* slots) {
    a = nh_wave_allreduce<nh_op_sum, 64>(a);
    b = nh_wave_allreduce<nh_op_sum, 64>(b);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slots[wave] = make_float2(a, b);
        __syncthreads();
        a = slots[0].x;
        b = slots[0].y;
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) {
            a += slots[w].x;
            b += slots[w].y;
        }
    }
}

template <typename T, int V> NEON_DEV void load_clipped(nh_raw<T, V>& r, const T* p, int n) {
    if (n >= V) r.load(p);
    else if (n > 0) r.load_partial(p, n);
    else r.zero();
}
template <typename T, int V> NEON_DEV void store_clipped(const nh_out<T, V>& o, T* p, int n, bool stream = false) {
    if (n >= V && stream) o.store_stream(p);
    else if (n >= V) o.store(p);
    else if (n > 0) o.store_partial(p, n);
}
// V fp32 values at p, the ones behind n zero
template <int V> NEON_DEV void load_floats(float (&f)[V], const float* p, int n) {
    if (n >= V) {
        nh_load_vec<float, V>(p, f);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = j < n ? p[j] : 0.0f;
    }
}
NEON_DEV int clip(long long left, int v) { return left >= v ? v : (left > 0 ? (int)left : 0); }

// Threads TPR per row (64: a wave, four rows per workgroup at a time).
template <int TPR> struct RowShape {
    static constexpr int NT = TPR == 64 ? 256 : TPR, RPB = TPR == 64 ? 4 : 1;
};

// ---------------------------------------------------------------------------
// rows, forward.  TPR threads hold one row in registers (NV 16-byte vectors
// each), so x is read once although the variance is taken around the mean.  A
// workgroup walks over rows with gamma and beta kept, and the next row is asked
// for before this one is summed up: loads return in the order of issue, stores
// among them, so a load behind this row's stores would wait for them.  The rows
// take turns in two sets of registers; moving the next row into this one's place
// would wait for it.  Bound by HBM: 16384 x 5000 bf16, 328 MB in 66 to 70 us (4.7 to 5.0
// TB/s; a workgroup per row 84 us, one set of registers 76 us).
// ---------------------------------------------------------------------------
template <typename T, int TPR, int NV> __global__ __launch_bounds__(RowShape<TPR>::NT) void ln_rows_fprop_kernel(LnArgs a) {
    constexpr int V = vec<T>::V, RPB = RowShape<TPR>::RPB;
    __shared__ float2 slots[2][TPR / 64];
    const int t = threadIdx.x % TPR;
    const float inv_f = 1.0f / (float)a.features;
    const size_t step = (size_t)gridDim.x * RPB;
    size_t row = (size_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (TPR == 64 && row >= a.positions) return;
    int n[NV];
    nh_raw<T, V> even[NV], odd[NV];
    const auto load = [&](nh_raw<T, V> (&to)[NV], size_t at) {
        const T* x = (const T*)a.x + at * a.ld_x;
#pragma unroll
        for (int k = 0; k < NV; ++k) load_clipped(to[k], x + (uint32_t)(k * TPR + t) * V, n[k]);
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) n[k] = clip((long long)a.features - (uint32_t)(k * TPR + t) * V, V);
    load(even, row);
    float g[NV][V], b[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        load_floats<V>(g[k], a.gamma + (uint32_t)(k * TPR + t) * V, n[k]);
        load_floats<V>(b[k], a.beta + (uint32_t)(k * TPR + t) * V, n[k]);
    }
    const auto normalise = [&](const nh_raw<T, V> (&r)[NV], size_t at) {
        float s = 0.0f, unused = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) s += r[k].get(j);
        row_sum2<TPR>(s, unused, slots[0]);
        const float mu = s * inv_f;
        float q = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = r[k].get(j) - mu;
                q = __builtin_fmaf(d, j < n[k] ? d : 0.0f, q);
            }
        }
        row_sum2<TPR>(q, unused, slots[1]);
        const float var = q * inv_f;
        const float rs = inv_std(var, a.eps);
        T* y = (T*)a.out + at * a.ld_out;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            nh_out<T, V> o;
            o.clear();
#pragma unroll
            for (int j = 0; j < V; ++j) o.set(j, __builtin_fmaf((r[k].get(j) - mu) * rs, g[k][j], b[k][j]));
            store_clipped(o, y + (uint32_t)(k * TPR + t) * V, n[k], a.stream);
        }
        if (t == 0) {
            a.mean[at] = mu;
            a.var[at] = var;
        }
    };
    for (;;) {
        if (row + step < a.positions) load(odd, row + step);
        normalise(even, row);
        row += step;
        if (row >= a.positions) return;
        if (row + step < a.positions) load(even, row + step);
        normalise(odd, row);
        row += step;
        if (row >= a.positions) return;
    }
}

// Rows of more features than that leaves registers for: one workgroup per row,
// gamma and beta read when they are needed.
template <typename T, int NV> __global__ __launch_bounds__(1024) void ln_rows_fprop_wide_kernel(LnArgs a) {
    constexpr int V = vec<T>::V, TPR = 1024;
    __shared__ float2 slots[2][TPR / 64];
    const size_t row = blockIdx.x;
    const int t = threadIdx.x;
    const T* x = (const T*)a.x + row * a.ld_x;
    T* y = (T*)a.out + row * a.ld_out;
    const float inv_f = 1.0f / (float)a.features;
    const auto left = [&](int k) { return clip((long long)a.features - (uint32_t)(k * TPR + t) * V, V); };
    nh_raw<T, V> r[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) load_clipped(r[k], x + (uint32_t)(k * TPR + t) * V, left(k));
    float s = 0.0f, unused = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) s += r[k].get(j);
        r[k].keep();
    }
    row_sum2<TPR>(s, unused, slots[0]);
    const float mu = s * inv_f;
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = r[k].get(j) - mu;
            q = __builtin_fmaf(d, j < left(k) ? d : 0.0f, q);
        }
        r[k].keep();
    }
    row_sum2<TPR>(q, unused, slots[1]);
    const float var = q * inv_f;
    const float rs = inv_std(var, a.eps);
    if (t == 0) {
        a.mean[row] = mu;
        a.var[row] = var;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t c = (uint32_t)(k * TPR + t) * V;
        const int n = left(k);
        float g[V], b[V];
        load_floats<V>(g, a.gamma + c, n);
        load_floats<V>(b, a.beta + c, n);
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int j = 0; j < V; ++j) o.set(j, __builtin_fmaf((r[k].get(j) - mu) * rs, g[j], b[j]));
        store_clipped(o, y + c, n);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// rows longer than the registers of a workgroup: three sweeps, the later two
// out of the caches
template <typename T> __global__ __launch_bounds__(1024) void ln_rows_fprop_long_kernel(LnArgs a) {
    constexpr int V = vec<T>::V;
    __shared__ float2 slots[2][16];
    const size_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.ld_x;
    T* y = (T*)a.out + row * a.ld_out;
    const float inv_f = 1.0f / (float)a.features;
    const long long F = a.features;
    float s = 0.0f, unused = 0.0f;
    for (long long c = (long long)threadIdx.x * V; c < F; c += 1024 * V) {
        nh_raw<T, V> r;
        load_clipped(r, x + c, clip(F - c, V));
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) v += r.get(j);
        s += v;
    }
    row_sum2<1024>(s, unused, slots[0]);
    const float mu = s * inv_f;
    float q = 0.0f;
    for (long long c = (long long)threadIdx.x * V; c < F; c += 1024 * V) {
        nh_raw<T, V> r;
        const int n = clip(F - c, V);
        load_clipped(r, x + c, n);
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = r.get(j) - mu;
            v = __builtin_fmaf(d, j < n ? d : 0.0f, v);
        }
        q += v;
    }
    row_sum2<1024>(q, unused, slots[1]);
    const float var = q * inv_f;
    const float rs = inv_std(var, a.eps);
    if (threadIdx.x == 0) {
        a.mean[row] = mu;
        a.var[row] = var;
    }
    for (long long c = (long long)threadIdx.x * V; c < F; c += 1024 * V) {
        nh_raw<T, V> r;
        const int n = clip(F - c, V);
        load_clipped(r, x + c, n);
        float g[V], b[V];
        load_floats<V>(g, a.gamma + c, n);
        load_floats<V>(b, a.beta + c, n);
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int j = 0; j < V; ++j) o.set(j, __builtin_fmaf((r.get(j) - mu) * rs, g[j], b[j]));
        store_clipped(o, y + c, n);
    }
}

// ---------------------------------------------------------------------------
// rows, backward: a workgroup walks over rows with a fixed set of features per
// thread, so the sums over positions for dgamma and dbeta stay in registers;
// each workgroup leaves one partial row of both (gridDim.x of them), which
// ln_param_kernel adds up in a fixed order.  Bound by HBM: 16384 x 2048 bf16, 201
// MB in 47 us (4.3 TB/s).  Rows that do not begin on 16 bytes cost about 1.7 times
// that per byte (7764 x 3356: 2.5 TB/s with the sum of the partial rows).
// ---------------------------------------------------------------------------
template <typename T, int TPR, int NV> __global__ __launch_bounds__(RowShape<TPR>::NT) void ln_rows_bprop_kernel(LnArgs a) {
    constexpr int V = vec<T>::V, RPB = RowShape<TPR>::RPB;
    __shared__ float2 slots[2][TPR / 64];
    const int t = threadIdx.x % TPR;
    const float inv_f = 1.0f / (float)a.features;
    const size_t step = (size_t)gridDim.x * RPB;
    size_t row = (size_t)blockIdx.x * RPB + threadIdx.x / TPR;
    int n[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) n[k] = clip((long long)a.features - (uint32_t)(k * TPR + t) * V, V);
    struct Row {
        nh_raw<T, V> x[NV], d[NV];
        float mean, var;
    };
    Row even, odd;
    const auto load = [&](Row& to, size_t at) {
        to.mean = a.mean[at];
        to.var = a.var[at];
        const T* x = (const T*)a.x + at * a.ld_x;
        const T* dy = (const T*)a.dy + at * a.ld_dy;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            load_clipped(to.x[k], x + (uint32_t)(k * TPR + t) * V, n[k]);
            load_clipped(to.d[k], dy + (uint32_t)(k * TPR + t) * V, n[k]);
        }
    };
    if (row < a.positions) load(even, row);
    float g[NV][V], dg[NV][V], db[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        load_floats<V>(g[k], a.gamma + (uint32_t)(k * TPR + t) * V, n[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) dg[k][j] = db[k][j] = 0.0f;
    }
    const auto go = [&](Row& r, size_t at, float2* slot) {
        const float mu = r.mean, rs = inv_std(r.var, a.eps);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (r.x[k].get(j) - mu) * rs, d = r.d[k].get(j), u = d * g[k][j];
                s1 += u;
                s2 = __builtin_fmaf(u, h, s2);
                dg[k][j] = __builtin_fmaf(d, h, dg[k][j]);
                db[k][j] += d;
            }
            // (widened again below)
            r.x[k].keep();
            r.d[k].keep();
        }
        row_sum2<TPR>(s1, s2, slot);
        s1 *= inv_f;
        s2 *= inv_f;
        T* dx = (T*)a.out + at * a.ld_out;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            nh_out<T, V> o;
            o.clear();
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (r.x[k].get(j) - mu) * rs, u = r.d[k].get(j) * g[k][j];
                o.set(j, rs * ((u - s1) - h * s2));
            }
            store_clipped(o, dx + (uint32_t)(k * TPR + t) * V, n[k], a.stream);
        }
    };
    // two sets of registers in turn, see the forward kernel -- where they fit
    if constexpr (TPR == 1024 && NV * V > 8) {
        for (int turn = 0; row < a.positions; turn ^= 1) {
            go(even, row, slots[turn]);
            row += step;
            if (row < a.positions) load(even, row);
        }
    } else {
        while (row < a.positions) {
            if (row + step < a.positions) load(odd, row + step);
            go(even, row, slots[0]);
            row += step;
            if (row >= a.positions) break;
            if (row + step < a.positions) load(even, row + step);
            go(odd, row, slots[1]);
            row += step;
        }
    }
    float* part = a.part + (size_t)blockIdx.x * 2 * a.features;
    if constexpr (TPR == 64) {
        // the four rows in flight of a workgroup: joined in wave order
        __shared__ float join[4][2][64 * V];
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) {
                join[wave][0][t * V + j] = dg[k][j];
                join[wave][1][t * V + j] = db[k][j];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * 64 * V; i += 256) {
                const int which = i / (64 * V), e = i % (64 * V);
                const uint32_t c = (uint32_t)k * 64 * V + e;
                if (c < a.features)
                    part[(size_t)which * a.features + c] =
                        ((join[0][which][e] + join[1][which][e]) + join[2][which][e]) + join[3][which][e];
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n[k]) {
                    const uint32_t c = (uint32_t)(k * TPR + t) * V + j;
                    part[c] = dg[k][j];
                    part[a.features + c] = db[k][j];
                }
    }
}

// rows too long for that: dx in two sweeps per row, the parameter sums by
// strips of features in a kernel of their own, so that x and dy are read three
// times, the third out of the caches in part: 4096 x 12000 fp32, 84 + 129 + 5 us for 590 MB that are
// needed, 1.34 GB moved (6.2 TB/s of those)
template <typename T> __global__ __launch_bounds__(1024) void ln_rows_bprop_long_kernel(LnArgs a) {
    constexpr int V = vec<T>::V;
    __shared__ float2 slots[16];
    const size_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.ld_x;
    const T* dy = (const T*)a.dy + row * a.ld_dy;
    T* dx = (T*)a.out + row * a.ld_out;
    const float inv_f = 1.0f / (float)a.features;
    const long long F = a.features;
    const float mu = a.mean[row], rs = inv_std(a.var[row], a.eps);
    float s1 = 0.0f, s2 = 0.0f;
    for (long long c = (long long)threadIdx.x * V; c < F; c += 1024 * V) {
        const int n = clip(F - c, V);
        nh_raw<T, V> rx, rd;
        float g[V];
        load_clipped(rx, x + c, n);
        load_clipped(rd, dy + c, n);
        load_floats<V>(g, a.gamma + c, n);
        float p1 = 0.0f, p2 = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float u = rd.get(j) * g[j];
            p1 += u;
            p2 = __builtin_fmaf(u, (rx.get(j) - mu) * rs, p2);
        }
        s1 += p1;
        s2 += p2;
    }
    row_sum2<1024>(s1, s2, slots);
    s1 *= inv_f;
    s2 *= inv_f;
    for (long long c = (long long)threadIdx.x * V; c < F; c += 1024 * V) {
        const int n = clip(F - c, V);
        nh_raw<T, V> rx, rd;
        float g[V];
        load_clipped(rx, x + c, n);
        load_clipped(rd, dy + c, n);
        load_floats<V>(g, a.gamma + c, n);
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int j = 0; j < V; ++j)
            o.set(j, rs * ((rd.get(j) * g[j] - s1) - ((rx.get(j) - mu) * rs) * s2));
        store_clipped(o, dx + c, n);
    }
}

// a wave per strip of 64 V features and run of `rows_per` rows (blockIdx.y)
template <typename T> __global__ __launch_bounds__(64) void ln_rows_params_kernel(LnArgs a, size_t rows_per) {
    constexpr int V = vec<T>::V;
    const long long c = ((long long)blockIdx.x * 64 + threadIdx.x) * V;
    const int n = clip((long long)a.features - c, V);
    if (n <= 0) return;
    const size_t r0 = (size_t)blockIdx.y * rows_per;
    const size_t r1 = r0 + rows_per < a.positions ? r0 + rows_per : a.positions;
    float dg[V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dg[j] = db[j] = 0.0f;
    for (size_t r = r0; r < r1; ++r) {
        nh_raw<T, V> rx, rd;
        load_clipped(rx, (const T*)a.x + r * a.ld_x + c, n);
        load_clipped(rd, (const T*)a.dy + r * a.ld_dy + c, n);
        const float mu = a.mean[r], rs = inv_std(a.var[r], a.eps);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = rd.get(j);
            dg[j] = __builtin_fmaf(d, (rx.get(j) - mu) * rs, dg[j]);
            db[j] += d;
        }
    }
    float* part = a.part + (size_t)blockIdx.y * 2 * a.features + c;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) {
            part[j] = dg[j];
            part[a.features + j] = db[j];
        }
}

// grads[which][f] = sum of `count` partial rows, in a fixed order: 128 threads
// per 4 features take every 128th row, joined in LDS.  Latency: 784 rows of 2 x 1024
// in 5 us (one thread per feature and 16th of the rows: 16 us).
__global__ __launch_bounds__(1024) void ln_param_kernel(LnArgs a, uint32_t count) {
    __shared__ float join[128][36];
    const int lane = threadIdx.x & 7, grp = threadIdx.x >> 3;
    const uint32_t f = blockIdx.x * 32 + lane * 4;
    const int n = clip((long long)a.features - f, 4);
    const float* p = a.part + (size_t)blockIdx.y * a.features + f;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n > 0) {
#pragma unroll 8
        for (uint32_t i = grp; i < count; i += 128) {
            float v[4];
            load_floats<4>(v, p + (size_t)i * 2 * a.features, n);
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += v[k];
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) join[grp][lane * 4 + k] = s[k];
    __syncthreads();
    // 32 threads per feature add 4 groups each, then the lanes
    const int c = threadIdx.x >> 5, part = threadIdx.x & 31;
    float r = ((join[part][c] + join[part + 32][c]) + join[part + 64][c]) + join[part + 96][c];
    r = nh_wave_allreduce<nh_op_sum, 32>(r);
    if (part == 0 && blockIdx.x * 32 + c < a.features) a.grads[blockIdx.y][blockIdx.x * 32 + c] = r;
}

// ---------------------------------------------------------------------------
// columns
// ---------------------------------------------------------------------------
// Strips dealt to the XCDs in contiguous runs: the two halves of a cache line
// that neighbouring strips of 64 bytes read meet in one L2.
NEON_DEV uint32_t strip_of_block() {
    const uint32_t n = gridDim.x, b = blockIdx.x, xcd = b % NH_XCDS, rest = n % NH_XCDS;
    return n < NH_XCDS ? b : xcd * (n / NH_XCDS) + (xcd < rest ? xcd : rest) + b / NH_XCDS;
}

// Running (mean, sum of squared deviations) of two disjoint sets of a column's
// values joined: with the counts the same for all columns a thread holds, the
// factors are computed once.  A side may be empty: its mean and m2 are 0.
struct JoinFactors {
    float to_b, cross;      // n_b / n and n_a n_b / n
    NEON_DEV JoinFactors(float na, float nb) {
        const float n = na + nb;
        to_b = n > 0.0f ? nb / n : 0.0f;
        cross = na * to_b;
    }
    // d * cross before the other d: of an empty side, where cross is 0 and d the other side's mean, nothing
    // is left whatever the square of d would be.  Where the difference is more than fp32 holds (an infinite
    // mean among them) the mean is added up from its parts, which leaves infinities what they are.
    NEON_DEV void join(float& mean, float& m2, float mean_b, float m2_b) const {
        const float d = mean_b - mean;
        const float parts = __builtin_fmaf(mean, 1.0f - to_b, mean_b * to_b);
        const float moved = __builtin_fmaf(d, to_b, mean);
        mean = fabsf(d) <= NH_FLT_MAX ? moved : parts;
        m2 = (m2 + m2_b) + (d * cross) * d;
    }
};

// Columns, forward: strips of LC lanes of 16 bytes of positions.  A thread holds
// V neighbouring columns and takes every (NT / LC)-th feature, RV at a time.
template <typename T, int NT, int LC, int RV> struct ColFprop {
    static constexpr int V = vec<T>::V, COLS = LC * V, NW = NT / 64, RL = NT / LC;
    struct Shared {
        float mean[NW][COLS], m2[NW][COLS], n[NW];
    };
    const LnArgs& a;
    uint32_t strip;
    int t, cl, rl, n;
    size_t c0, c;
    nh_raw<T, V> r[RV];
    float g[RV], b[RV];
    float mean[V], m2[V], count;

    NEON_DEV ColFprop(const LnArgs& args, uint32_t strip_) : a(args), strip(strip_) {
        t = threadIdx.x;
        cl = t % LC;
        rl = t / LC;
        c0 = (size_t)strip * COLS;
        c = c0 + cl * V;
        n = clip((long long)a.positions - (long long)c, V);
        count = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.0f;
    }
    // features base + rl + i RL below `end` (the last one again behind it)
    NEON_DEV void load_params(uint32_t base, uint32_t end) {
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const uint32_t f = base + rl + i * RL < end ? base + rl + i * RL : end - 1;
            g[i] = a.gamma[f];
            b[i] = a.beta[f];
        }
    }
    NEON_DEV void load(uint32_t base, uint32_t end) {
        const T* x = (const T*)a.x + c;
        if (c0 + COLS <= a.positions) {
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + rl + i * RL < end ? base + rl + i * RL : end - 1;
                r[i].load(x + (size_t)f * a.ld_x);
            }
        } else {
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + rl + i * RL < end ? base + rl + i * RL : end - 1;
                load_clipped(r[i], x + (size_t)f * a.ld_x, n);
            }
        }
    }
    // FIRST: there is nothing to join them with
    template <bool FIRST> NEON_DEV void add(uint32_t base, uint32_t end) {
        int rows = 0;
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            if (base + rl + i * RL < end) ++rows;
            else r[i].zero();
        }
        const JoinFactors jf(count, (float)rows);
        const float inv = rows > 0 ? 1.0f / (float)rows : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < RV; ++i) s += r[i].get(j);
            const float m = s * inv;
            float q = 0.0f;
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const float d = r[i].get(j) - m;
                q = __builtin_fmaf(d, i < rows ? d : 0.0f, q);
            }
            if constexpr (FIRST) {
                mean[j] = m;
                m2[j] = q;
            } else {
                jf.join(mean[j], m2[j], m, q);
            }
        }
        count += (float)rows;
        // (widened again when they are used next: kept as floats they take twice the registers)
#pragma unroll
        for (int i = 0; i < RV; ++i) r[i].keep();
    }
    template <int X> NEON_DEV void fold() {
        if constexpr (X < 64) {
            // Each side by its share: commutative, so that both partners get the same bits.  The shares are
            // mostly halves, with which the mean is rounded once; an infinite mean stays one.
            const float nb = nh_lane_xor<X>(count), n = count + nb;
            const float mine = n > 0.0f ? count / n : 0.0f, other = n > 0.0f ? nb / n : 0.0f;
            const float cross = n * (mine * other);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float om = nh_lane_xor<X>(mean[j]), oq = nh_lane_xor<X>(m2[j]), d = om - mean[j];
                mean[j] = mean[j] * mine + om * other;
                m2[j] = (m2[j] + oq) + (d * cross) * d;
            }
            count += nb;
            fold<2 * X>();
        }
    }
    // lanes of a wave that share columns, then the waves: thread t < COLS gets column t's
    NEON_DEV float2 join(Shared& m) {
        fold<LC>();
        const int wave = t >> 6;
        if ((t & 63) < LC) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                m.mean[wave][cl * V + j] = mean[j];
                m.m2[wave][cl * V + j] = m2[j];
            }
            if (cl == 0) m.n[wave] = count;
        }
        __syncthreads();
        float2 r = make_float2(0.0f, 0.0f);
        if (t < COLS) {
            r = make_float2(m.mean[0][t], m.m2[0][t]);
            float k = m.n[0];
            for (int w = 1; w < NW; ++w) {
                JoinFactors(k, m.n[w]).join(r.x, r.y, m.mean[w][t], m.m2[w][t]);
                k += m.n[w];
            }
        }
        return r;
    }
    // thread t < COLS has column t's finished pair: mean and 1 / std for every thread's columns
    NEON_DEV void share(Shared& m, float2 r, bool keep) {
        const float inv_f = 1.0f / (float)a.features;
        if (t < COLS) {
            const float var = r.y * inv_f;
            m.mean[0][t] = r.x;
            m.m2[0][t] = inv_std(var, a.eps);
            if (keep && c0 + t < a.positions) {
                a.mean[c0 + t] = r.x;
                a.var[c0 + t] = var;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) {
            mean[j] = m.mean[0][cl * V + j];
            m2[j] = m.m2[0][cl * V + j];
        }
    }
    NEON_DEV void put(uint32_t base, uint32_t end) {
        T* y = (T*)a.out + c;
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const uint32_t f = base + rl + i * RL;
            if (f >= end) continue;
            nh_out<T, V> o;
            o.clear();
#pragma unroll
            for (int j = 0; j < V; ++j) o.set(j, __builtin_fmaf((r[i].get(j) - mean[j]) * m2[j], g[i], b[i]));
            store_clipped(o, y + (size_t)f * a.ld_out, n);
        }
    }
};

// The features of a strip in registers: x is read once.  Loads return in the
// order of issue, stores among them, so gamma and beta are asked for first.
// 1024 x 25088 fp16, 103 MB: 31 us (3.3 TB/s); in the two-pass form below 33-39 us.
// Bound by the 64-byte pieces of 50 KB lines.
template <typename T, int NT, int LC, int RV> __global__ __launch_bounds__(NT, 4) void ln_cols_fprop_kernel(LnArgs a) {
    using K = ColFprop<T, NT, LC, RV>;
    __shared__ typename K::Shared m;
    K k(a, strip_of_block());
    k.load_params(0, a.features);
    k.load(0, a.features);
    k.template add<true>(0, a.features);
    k.share(m, k.join(m), true);
    k.put(0, a.features);
}

// More features than that: statistics of runs of features (blockIdx.y), then the
// runs' statistics joined in order by every workgroup that finishes one.  x is read
// twice: 4096 x 16384 bf16, 38 + 59 us for 269 MB that are needed, 414 moved (4.2 TB/s of those).
template <typename T> __global__ __launch_bounds__(256) void ln_cols_fprop_sums_kernel(LnArgs a, uint32_t rows_per, uint32_t chunks,
                                                                                      float2* sums) {
    using K = ColFprop<T, 256, 8, 8>;
    __shared__ typename K::Shared m;
    K k(a, strip_of_block());
    const uint32_t r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < a.features ? r0 + rows_per : a.features;
    k.load(r0, r1);
    k.template add<true>(r0, r1);
    for (uint32_t base = r0 + K::RL * 8; base < r1; base += K::RL * 8) {
        k.load(base, r1);
        k.template add<false>(base, r1);
    }
    const float2 r = k.join(m);
    if (k.t < K::COLS) sums[((size_t)k.strip * chunks + blockIdx.y) * K::COLS + k.t] = r;
}
template <typename T> __global__ __launch_bounds__(256) void ln_cols_fprop_finish_kernel(LnArgs a, uint32_t rows_per, uint32_t chunks,
                                                                                        const float2* sums) {
    using K = ColFprop<T, 256, 8, 8>;
    __shared__ typename K::Shared m;
    K k(a, strip_of_block());
    const uint32_t r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < a.features ? r0 + rows_per : a.features;
    k.load_params(r0, r1);
    k.load(r0, r1);
    float2 r = make_float2(0.0f, 0.0f);
    if (k.t < K::COLS) {
        float seen = 0.0f;
        for (uint32_t i = 0; i < chunks; ++i) {
            const float2 p = sums[((size_t)k.strip * chunks + i) * K::COLS + k.t];
            const uint32_t b = i * rows_per, e = b + rows_per < a.features ? b + rows_per : a.features;
            JoinFactors(seen, (float)(e - b)).join(r.x, r.y, p.x, p.y);
            seen += (float)(e - b);
        }
    }
    k.share(m, r, blockIdx.y == 0);
    for (uint32_t base = r0; base < r1; base += K::RL * 8) {
        if (base != r0) {
            k.load_params(base, r1);
            k.load(base, r1);
        }
        k.put(base, r1);
    }
}

// Columns, backward: strips of 64 bytes of positions (4 lanes of 16 bytes).  A
// thread holds V neighbouring columns and takes every (NT / 4)-th feature.
constexpr int BLC = 4;
template <typename T> struct bstrip { static constexpr int COLS = BLC * vec<T>::V; };

template <typename T, int NT> struct ColBprop {
    static constexpr int V = vec<T>::V, COLS = bstrip<T>::COLS, NW = NT / 64, RL = NT / BLC;
    struct Shared {
        float a[NW][COLS], b[NW][COLS];
    };
    const LnArgs& a;
    uint32_t strip;
    int t, cl, rl, n;
    size_t c0, c;
    const T* x;
    const T* dy;
    float mu[V], rs[V], s1[V], s2[V];

    NEON_DEV ColBprop(const LnArgs& args, uint32_t strip_) : a(args), strip(strip_) {
        t = threadIdx.x;
        cl = t % BLC;
        rl = t / BLC;
        c0 = (size_t)strip * COLS;
        c = c0 + cl * V;
        n = clip((long long)a.positions - (long long)c, V);
        x = (const T*)a.x + c;
        dy = (const T*)a.dy + c;
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
    }
    NEON_DEV void load_stats() {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            mu[j] = j < n ? a.mean[c + j] : 0.0f;
            rs[j] = j < n ? inv_std(a.var[c + j], a.eps) : 0.0f;
        }
    }
    // one feature's share of the column sums; returns the feature's sums over the strip
    NEON_DEV float2 add(const nh_raw<T, V>& rx, const nh_raw<T, V>& rd, float g) {
        float dg = 0.0f, db = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            // (the deviation is normalised first: its product with the error may leave fp32 without that)
            const float d = rd.get(j), e = (rx.get(j) - mu[j]) * rs[j] * d;
            s1[j] = __builtin_fmaf(d, g, s1[j]);
            s2[j] = __builtin_fmaf(e, g, s2[j]);
            dg += e;
            db += d;
        }
        // (the sums are in registers here: left to itself the compiler puts these additions off until
        // they are read, and keeps every h and d for them)
#pragma unroll
        for (int j = 0; j < V; ++j) asm volatile("" : "+v"(s1[j]), "+v"(s2[j]));
        return make_float2(nh_wave_allreduce<nh_op_sum, BLC>(dg), nh_wave_allreduce<nh_op_sum, BLC>(db));
    }
    NEON_DEV void put_sums(uint32_t f, float2 r) {
        float* part = a.part + (size_t)strip * 2 * a.features;
        part[f] = r.x;
        part[a.features + f] = r.y;
    }
    NEON_DEV void put(const nh_raw<T, V>& rx, const nh_raw<T, V>& rd, float g, uint32_t f) {
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int j = 0; j < V; ++j) {
            // s1, s2 as share() leaves them: r mean(u), r mean(u h)
            const float u = __builtin_fmaf(rd.get(j) * rs[j], g, -s1[j]);
            o.set(j, __builtin_fmaf(-s2[j], (rx.get(j) - mu[j]) * rs[j], u));
        }
        store_clipped(o, (T*)a.out + c + (size_t)f * a.ld_out, n);
    }
    // features [r0, r1) straight from memory, a few at a time
    template <int RV, class F> NEON_DEV void stream(uint32_t r0, uint32_t r1, F each) {
        const bool full = c0 + COLS <= a.positions;
        for (uint32_t base = r0 + rl; base - rl < r1; base += RL * RV) {
            nh_raw<T, V> rx[RV], rd[RV];
            float g[RV];
#pragma unroll
            for (int i = 0; i < RV; ++i) g[i] = a.gamma[base + i * RL < r1 ? base + i * RL : r1 - 1];
            if (full) {
#pragma unroll
                for (int i = 0; i < RV; ++i) {
                    const uint32_t f = base + i * RL < r1 ? base + i * RL : r1 - 1;
                    rx[i].load(x + (size_t)f * a.ld_x);
                    rd[i].load(dy + (size_t)f * a.ld_dy);
                }
            } else {
#pragma unroll
                for (int i = 0; i < RV; ++i) {
                    const uint32_t f = base + i * RL < r1 ? base + i * RL : r1 - 1;
                    load_clipped(rx[i], x + (size_t)f * a.ld_x, n);
                    load_clipped(rd[i], dy + (size_t)f * a.ld_dy, n);
                }
            }
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + i * RL;
                if (f >= r1) {       // (a feature once more: no error, no share)
                    rx[i].zero();
                    rd[i].zero();
                }
                each(rx[i], rd[i], g[i], f, f < r1);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    // column sums over the 16 lanes of a wave that share columns and over the waves:
    // thread t < COLS gets column t's
    NEON_DEV float2 join(Shared& m) {
        const int j = nh_col_wave_fold<nh_op_sum, V, BLC>(s1);
        nh_col_wave_fold<nh_op_sum, V, BLC>(s2);
        constexpr int LEFT = V * BLC / 64 > 1 ? V * BLC / 64 : 1;      // columns a lane is left with
#pragma unroll
        for (int i = 0; i < LEFT; ++i) {
            m.a[t >> 6][cl * V + j + i] = s1[i];
            m.b[t >> 6][cl * V + j + i] = s2[i];
        }
        __syncthreads();
        float2 r = make_float2(0.0f, 0.0f);
        if (t < COLS)
            for (int w = 0; w < NW; ++w) {
                r.x += m.a[w][t];
                r.y += m.b[w][t];
            }
        return r;
    }
    // thread t < COLS has the finished sums of column t: means for every thread's columns
    NEON_DEV void share(Shared& m, float2 r) {
        const float inv_f = 1.0f / (float)a.features;
        if (t < COLS) {
            m.a[0][t] = r.x * inv_f;
            m.b[0][t] = r.y * inv_f;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s1[j] = m.a[0][cl * V + j] * rs[j];
            s2[j] = m.b[0][cl * V + j] * rs[j];
        }
    }
};

// The features of a strip in registers (RV per thread): x and dy are read once.
// The strip that the positions end in streams them twice instead.
//
// Loads return in the order of issue, stores among them: what is small (the
// statistics, gamma) is asked for first, the features' sums go through LDS and
// are stored last, so that the additions of a feature wait for its own two loads
// only.  1024 x 25088 fp16, 154 MB: 53 us (2.9 TB/s); with gamma read where it is
// used and the sums stored at once 65 us, with both tensors streamed twice 58-60
// us.  What is left: 784 strips on 512 places, and lines of 50 KB of which a strip
// reads 64 bytes.
template <typename T, int NT, int RV> __global__ __launch_bounds__(NT, 4) void ln_cols_bprop_kernel(LnArgs a) {
    using K = ColBprop<T, NT>;
    __shared__ typename K::Shared m;
    __shared__ float2 feature[K::RL * RV];
    K k(a, strip_of_block());
    const uint32_t last = a.features - 1;
    if (k.c0 + K::COLS <= a.positions) {
        k.load_stats();
        nh_raw<T, K::V> rx[RV], rd[RV];
        float g[RV];
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const uint32_t f = k.rl + i * K::RL;
            g[i] = a.gamma[f < last ? f : last];
        }
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const uint32_t f = k.rl + i * K::RL < last ? k.rl + i * K::RL : last;
            rx[i].load(k.x + (size_t)f * a.ld_x);
            rd[i].load(k.dy + (size_t)f * a.ld_dy);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const uint32_t f = k.rl + i * K::RL;
            if (f > last) {       // (a feature once more: no error, no share)
                rx[i].zero();
                rd[i].zero();
            }
            const float2 r = k.add(rx[i], rd[i], g[i]);
            if (k.cl == 0) feature[f] = r;
            // the packed values are widened again below: kept as floats, or with the rows
            // interleaved, two tensors do not fit 128 registers
            rx[i].keep();
            rd[i].keep();
            __builtin_amdgcn_sched_barrier(0);
        }
        k.share(m, k.join(m));
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const uint32_t f = k.rl + i * K::RL;
            if (f <= last) k.put(rx[i], rd[i], g[i], f);
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
        k.load_stats();
        k.template stream<2>(0, a.features, [&](const auto& rx, const auto& rd, float g, uint32_t f, bool on) {
            const float2 r = k.add(rx, rd, g);
            if (k.cl == 0 && on) feature[f] = r;
        });
        k.share(m, k.join(m));
        k.template stream<2>(0, a.features, [&](const auto& rx, const auto& rd, float g, uint32_t f, bool on) {
            if (on) k.put(rx, rd, g, f);
        });
    }
    for (uint32_t f = threadIdx.x; f <= last; f += NT) k.put_sums(f, feature[f]);
}

// More features than that: column sums of runs of features (blockIdx.y), then
// the runs' sums joined in order by every workgroup that finishes one.  x and dy
// are read twice: 4096 x 16384 bf16, 72 + 87 + 6 us for 403 MB that are needed, 742 moved (4.5
// TB/s of those).
template <typename T> __global__ __launch_bounds__(256) void ln_cols_bprop_sums_kernel(LnArgs a, uint32_t rows_per, uint32_t chunks,
                                                                                      float2* sums) {
    using K = ColBprop<T, 256>;
    __shared__ typename K::Shared m;
    K k(a, strip_of_block());
    const uint32_t r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < a.features ? r0 + rows_per : a.features;
    k.load_stats();
    k.template stream<2>(r0, r1, [&](const auto& rx, const auto& rd, float g, uint32_t f, bool on) {
        const float2 r = k.add(rx, rd, g);
        if (k.cl == 0 && on) k.put_sums(f, r);
    });
    const float2 r = k.join(m);
    if (k.t < K::COLS) sums[((size_t)k.strip * chunks + blockIdx.y) * K::COLS + k.t] = r;
}
template <typename T> __global__ __launch_bounds__(256) void ln_cols_bprop_finish_kernel(LnArgs a, uint32_t rows_per, uint32_t chunks,
                                                                                        const float2* sums) {
    using K = ColBprop<T, 256>;
    __shared__ typename K::Shared m;
    K k(a, strip_of_block());
    const uint32_t r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < a.features ? r0 + rows_per : a.features;
    k.load_stats();
    float2 r = make_float2(0.0f, 0.0f);
    if (k.t < K::COLS)
        for (uint32_t i = 0; i < chunks; ++i) {
            const float2 p = sums[((size_t)k.strip * chunks + i) * K::COLS + k.t];
            r.x += p.x;
            r.y += p.y;
        }
    k.share(m, r);
    k.template stream<2>(r0, r1, [&](const auto& rx, const auto& rd, float g, uint32_t f, bool on) {
        if (on) k.put(rx, rd, g, f);
    });
}

// ---------------------------------------------------------------------------
// launch geometry
// ---------------------------------------------------------------------------
// features one workgroup's registers hold; with twice as many fp32 ones 20 registers spill, and
// the three sweeps are as fast or faster over most of that range: 200 x 33000 17.3 us against
// 21.4, 2000 x 40000 197 against 216, 5000 x 50000 592 both, 1000 x 65536 168 against 156
size_t long_row_fprop(int dtype) { return dtype == NH_T_F32 ? 32768 : 65536; }
// features of a row that the backward kernel holds with its parameter sums (16 fp32 features
// per thread of 1024 spill 61 registers)
size_t long_row_bprop(int dtype) { return dtype == NH_T_F32 ? 8192 : 16384; }
// Workgroups that walk over rows.  Forward, threads per CU (us with 1024, 2048): 16384 x 5000 bf16 67.8,
// 68.1; 46000 x 1500 fp32 106, 109; 4096 x 4096 fp32 26.0, 27.5; and the other way 100000 x 100 fp32 19.9,
// 17.7; 3000 x 600 fp32 6.4, 5.8 (512: 97, 109, 29, 28, 8).
// Backward, where every workgroup leaves a partial row of both parameter sums (us with 256, 512, 1024
// workgroups, their sum included): 16384 x 2048 bf16 73.6, 51.4, 52.0; 65536 x 768 bf16 87.2, 62.5, 69.2;
// 8000 x 4000 fp32 74.6, 78.5, 86.7.
constexpr size_t FPROP_THREADS = 2048;
constexpr size_t BPROP_BLOCKS = 512;
// Rows at least that a workgroup leaves one partial row for (us with 1, 3, 6): 777 x 1537 fp32 14.4, 12.0,
// 14.8; 512 x 4096 bf16 24.0, 16.3, 17.2; 2048 x 1024 bf16 11.1, 10.7, 14.9.
constexpr size_t BPROP_ROWS = 3;
constexpr size_t STREAM_BYTES = (size_t)256 << 20;           // what the last-level cache holds
constexpr unsigned LONG_ROW_RUNS = 64;        // row runs per feature strip in ln_rows_params_kernel
constexpr size_t COL_CHUNKS = 32;             // runs of tiles per strip of a split column kernel, at most

// forward and backward column kernels: features of one tile of the split form, features that stay in registers
struct ColLimits {
    size_t tile, resident, bytes;             // bytes: width of a strip
};
constexpr ColLimits COL_FPROP = {256, 2048, 128}, COL_BPROP = {512, 2048, 64};

size_t strips_of(const ColLimits& l, int dtype, size_t positions) { return lm::ceil_div(positions, l.bytes / lm::item_bytes(dtype)); }

struct ColSplit {
    uint32_t rows_per, chunks;
};
ColSplit split_columns(const ColLimits& l, size_t features) {
    const size_t tiles = lm::ceil_div(features, l.tile);
    const size_t per = lm::ceil_div(tiles, COL_CHUNKS);
    return {(uint32_t)(per * l.tile), (uint32_t)lm::ceil_div(tiles, per)};
}

// workgroups that walk over rows with `threads` each per row
unsigned row_blocks(size_t positions, size_t threads, size_t per_cu) {
    const size_t rows = threads == 64 ? 4 : 1, most = 256 * per_cu / (threads == 64 ? 256 : threads);
    const size_t blocks = lm::ceil_div(positions, rows);
    return (unsigned)(blocks < most ? blocks : most);
}
// Threads per row of the backward kernel: 8 features each (16 where a wave or a whole workgroup takes the
// row).  8000 x 4000 fp32 80 us, 8903 x 5610 bf16 109 us; with 16 each on half the threads, 165 registers
// leave two workgroups per CU and the latter took 181 us.
size_t bprop_threads(size_t features) { return features <= 64 * 16 ? 64 : features <= 256 * 8 ? 256 : features <= 512 * 8 ? 512 : 1024; }
unsigned bprop_blocks(size_t features, size_t positions) {
    const size_t threads = bprop_threads(features), rows = threads == 64 ? 4 : 1;
    // (two workgroups of 1024 threads do not fit a CU)
    const size_t most = threads == 1024 ? BPROP_BLOCKS / 2 : BPROP_BLOCKS;
    const size_t blocks = lm::ceil_div(positions, rows * BPROP_ROWS);
    return (unsigned)(blocks < most ? blocks : most);
}

size_t partial_rows(size_t features, size_t positions, int dtype, bool columns) {
    if (columns) return strips_of(COL_BPROP, dtype, positions);
    if (features > long_row_bprop(dtype)) return positions < LONG_ROW_RUNS ? positions : LONG_ROW_RUNS;
    return bprop_blocks(features, positions);
}

size_t column_sum_bytes(const ColLimits& l, size_t features, size_t positions, int dtype) {
    if (features <= l.resident) return 0;
    return lm::align256(strips_of(l, dtype, positions) * split_columns(l, features).chunks * (l.bytes / lm::item_bytes(dtype)) *
                        2 * sizeof(float));
}

size_t workspace_bytes(bool backward, int dtype, bool columns, size_t features, size_t positions) {
    if (!backward) return columns ? column_sum_bytes(COL_FPROP, features, positions, dtype) : 0;
    return (columns ? column_sum_bytes(COL_BPROP, features, positions, dtype) : 0) +
           lm::align256(partial_rows(features, positions, dtype, columns) * 2 * features * sizeof(float));
}

int check(const char* who, int dtype, int axis, size_t features, size_t positions, size_t ld_min_a, size_t ld_min_b,
          size_t ld_min_c) {
    if (!lm::known_dtype(dtype)) return lm::refuse(who, "unknown storage type");
    if (axis != 0 && axis != 1) return lm::refuse(who, "axis is 0 or 1");
    if (features == 0 || features > 0x7FFFFFFF) return lm::refuse(who, "between 1 and 2^31 - 1 features");
    if (positions > (size_t)1 << 40) return lm::refuse(who, "more than 2^40 positions");
    const size_t len = axis == 1 ? features : positions, lines = axis == 1 ? positions : features;
    if (lines > 1 && (ld_min_a < len || ld_min_b < len || ld_min_c < len))
        return lm::refuse(who, "leading dimension shorter than a line");
    return 0;
}

template <typename T> constexpr int code_of() { return sizeof(T) == 4 ? NH_T_F32 : NH_T_F16; }     // (as far as sizes go)

template <typename T> void fprop_rows(const LnArgs& a, lm::Launches& launch) {
    constexpr size_t V = vec<T>::V;
    const size_t nvec = lm::ceil_div(a.features, V);
    if (a.features > long_row_fprop(code_of<T>())) return launch(ln_rows_fprop_long_kernel<T>, a.positions, 1, 1024, 0, a);
#define LN_WIDE(NV) launch(ln_rows_fprop_wide_kernel<T, NV>, a.positions, 1, 1024, 0, a)
#define LN_GO(TPR, NV) launch(ln_rows_fprop_kernel<T, TPR, NV>, row_blocks(a.positions, TPR, FPROP_THREADS), 1, RowShape<TPR>::NT, 0, a)
    if (nvec <= 64) LN_GO(64, 1);
    else if (nvec <= 128) LN_GO(64, 2);
    else if (nvec <= 256) LN_GO(256, 1);
    else if (nvec <= 512) LN_GO(256, 2);
    else if (nvec <= 1024) LN_GO(512, 2);
    else if (nvec <= 2048) LN_GO(1024, 2);
    else if (nvec <= 4096) LN_WIDE(4);
    else LN_WIDE(8);
#undef LN_WIDE
#undef LN_GO
}

template <typename T> void fprop_cols(const LnArgs& a, lm::Launches& launch) {
#define LN_GO(NT, LC) launch(ln_cols_fprop_kernel<T, NT, LC, 8>, lm::ceil_div(a.positions, (LC) * vec<T>::V), 1, NT, 0, a)
    // strips of 128 bytes where four workgroups of them fit a CU (256 x 100352 fp16: 26.1 us, of 64 bytes 30.1;
    // 200 x 25088 bf16 8.8 and 10.9; 256 x 1024 fp32 4.8 and 4.7; 256 x 128 fp32, four workgroups or eight, 4.2
    // and 4.5), else of 64 (700 x 50000 fp32: 69 us, of 128 bytes and 1024 threads 79.7)
    if (a.features <= COL_FPROP.tile) {
        LN_GO(256, 8);
    } else if (a.features <= 1024) {
        LN_GO(512, 4);
    } else if (a.features <= COL_FPROP.resident) {
        LN_GO(1024, 4);
    } else {
        const size_t strips = strips_of(COL_FPROP, code_of<T>(), a.positions);
        const ColSplit c = split_columns(COL_FPROP, a.features);
        float2* sums = (float2*)a.part;
        launch(ln_cols_fprop_sums_kernel<T>, strips, c.chunks, 256, 0, a, c.rows_per, c.chunks, sums);
        launch(ln_cols_fprop_finish_kernel<T>, strips, c.chunks, 256, 0, a, c.rows_per, c.chunks, sums);
    }
#undef LN_GO
}

void add_params(const LnArgs& a, size_t count, lm::Launches& launch) {
    launch(ln_param_kernel, lm::ceil_div(a.features, 32), 2, 1024, 0, a, count);
}

template <typename T> void bprop_rows(const LnArgs& a, lm::Launches& launch) {
    constexpr size_t V = vec<T>::V;
    const size_t rows = partial_rows(a.features, a.positions, code_of<T>(), false);
    if (a.features > long_row_bprop(code_of<T>())) {
        const size_t per = lm::ceil_div(a.positions, rows), nvec = lm::ceil_div(a.features, V);
        // (the sums first: dx may take the place of dy)
        launch(ln_rows_params_kernel<T>, lm::ceil_div(nvec, 64), (unsigned)rows, 64, 0, a, per);
        launch(ln_rows_bprop_long_kernel<T>, a.positions, 1, 1024, 0, a);
        return add_params(a, rows, launch);
    }
#define LN_GO(TPR, NV) launch(ln_rows_bprop_kernel<T, TPR, NV>, rows, 1, RowShape<TPR>::NT, 0, a)
    if (a.features <= 64 * V) LN_GO(64, 1);
    else if (a.features <= 64 * 8) LN_GO(64, 8 / V < 2 ? 1 : 2);
    else if (a.features <= 64 * 16) LN_GO(64, 16 / V);
    else if (a.features <= 256 * 8) LN_GO(256, 8 / V);
    else if (a.features <= 512 * 8) LN_GO(512, 8 / V);
    else if (a.features <= 1024 * 8) LN_GO(1024, 8 / V);
    else if constexpr (sizeof(T) == 2) LN_GO(1024, 16 / V);
#undef LN_GO
    add_params(a, rows, launch);
}

template <typename T> void bprop_cols(LnArgs a, char* ws, lm::Launches& launch) {
    const size_t strips = strips_of(COL_BPROP, code_of<T>(), a.positions);
    float2* sums = (float2*)ws;
    a.part = (float*)(ws + column_sum_bytes(COL_BPROP, a.features, a.positions, code_of<T>()));
    if (a.features <= 512) {
        launch(ln_cols_bprop_kernel<T, 256, 8>, strips, 1, 256, 0, a);
    } else if (a.features <= 1024) {
        launch(ln_cols_bprop_kernel<T, 512, 8>, strips, 1, 512, 0, a);
    } else if (a.features <= COL_BPROP.resident) {
        launch(ln_cols_bprop_kernel<T, 1024, 8>, strips, 1, 1024, 0, a);
    } else {
        const ColSplit c = split_columns(COL_BPROP, a.features);
        launch(ln_cols_bprop_sums_kernel<T>, strips, c.chunks, 256, 0, a, c.rows_per, c.chunks, sums);
        launch(ln_cols_bprop_finish_kernel<T>, strips, c.chunks, 256, 0, a, c.rows_per, c.chunks, sums);
    }
    add_params(a, strips, launch);
}

}  // namespace

extern "C" {

size_t nh_ln_workspace_bytes(int backward, int dtype, int axis, size_t features, size_t positions) {
    if (!lm::known_dtype(dtype) || (axis != 0 && axis != 1)) return 0;
    return workspace_bytes(backward != 0, dtype, axis == 0, features, positions);
}

int nh_ln_fprop(void* y, float* mean, float* var, const void* x, const float* gamma, const float* beta, float eps, int dtype,
                int axis, size_t features, size_t positions, size_t ld_x, size_t ld_y, void* workspace,
                size_t workspace_bytes_given, void* stream) {
    if (int rc = check("nh_ln_fprop", dtype, axis, features, positions, ld_x, ld_y, ld_y)) return rc;
    if (positions == 0) return 0;
    if (!y || !mean || !var || !x || !gamma || !beta) return lm::refuse("nh_ln_fprop", "null pointer");
    const size_t need = workspace_bytes(false, dtype, axis == 0, features, positions);
    if (need && (!workspace || workspace_bytes_given < need))
        return lm::refuse("nh_ln_fprop", "workspace smaller than nh_ln_workspace_bytes");
    if (!lm::aligned16(workspace)) return lm::refuse("nh_ln_fprop", "workspace off a 16-byte boundary");
    LnArgs a = {};
    a.x = x; a.out = y; a.gamma = gamma; a.beta = beta; a.mean = mean; a.var = var; a.part = (float*)workspace;
    a.eps = eps; a.features = (uint32_t)features; a.positions = positions; a.ld_x = ld_x; a.ld_out = ld_y;
    a.stream = 2 * features * positions * lm::item_bytes(dtype) >= STREAM_BYTES;
    return lm::run("nh_ln_fprop", stream, [&](lm::Launches& launch) {
        lm::by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            axis == 1 ? fprop_rows<T>(a, launch) : fprop_cols<T>(a, launch);
        });
    });
}

int nh_ln_bprop(void* dx, float* dgamma, float* dbeta, const void* dy, const void* x, const float* mean, const float* var,
                const float* gamma, float eps, int dtype, int axis, size_t features, size_t positions, size_t ld_x,
                size_t ld_dy, size_t ld_dx, void* workspace, size_t workspace_bytes_given, void* stream) {
    if (int rc = check("nh_ln_bprop", dtype, axis, features, positions, ld_x, ld_dy, ld_dx)) return rc;
    if (!dgamma || !dbeta || !gamma) return lm::refuse("nh_ln_bprop", "null pointer");
    if (positions && (!dx || !dy || !x || !mean || !var)) return lm::refuse("nh_ln_bprop", "null pointer");
    const size_t need = workspace_bytes(true, dtype, axis == 0, features, positions);
    if (need && (!workspace || workspace_bytes_given < need))
        return lm::refuse("nh_ln_bprop", "workspace smaller than nh_ln_workspace_bytes");
    if (!lm::aligned16(workspace)) return lm::refuse("nh_ln_bprop", "workspace off a 16-byte boundary");
    LnArgs a = {};
    a.x = x; a.dy = dy; a.out = dx; a.gamma = gamma; a.mean = const_cast<float*>(mean); a.var = const_cast<float*>(var);
    a.part = (float*)workspace; a.grads[0] = dgamma; a.grads[1] = dbeta;
    a.eps = eps; a.features = (uint32_t)features; a.positions = positions; a.ld_x = ld_x; a.ld_dy = ld_dy; a.ld_out = ld_dx;
    a.stream = 3 * features * positions * lm::item_bytes(dtype) >= STREAM_BYTES;
    return lm::run("nh_ln_bprop", stream, [&](lm::Launches& launch) {
        if (positions == 0) return add_params(a, 0, launch);          // sums over no positions
        lm::by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            axis == 1 ? bprop_rows<T>(a, launch) : bprop_cols<T>(a, (char*)workspace, launch);
        });
    });
}

}  // extern "C"
