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
};

NEON_DEV float inv_std(float var, float eps) { return 1.0f / sqrtf(var + eps); }

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
template <typename T, int V> NEON_DEV void store_clipped(const nh_out<T, V>& o, T* p, int n) {
    if (n >= V) o.store(p);
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

// ---------------------------------------------------------------------------
// rows, forward: TPR threads hold one row in registers (NV 16-byte vectors
// each), so x is read once although the variance is taken around the mean.
// ---------------------------------------------------------------------------
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void ln_rows_fprop_kernel(LnArgs a) {
    constexpr int V = vec<T>::V;
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float2 slots[2][TPR / 64];
    const size_t row = (size_t)blockIdx.x * RPB + threadIdx.x / TPR;
    const int t = threadIdx.x % TPR;
    if (TPR == 64 && row >= a.positions) return;
    const T* x = (const T*)a.x + row * a.ld_x;
    T* y = (T*)a.out + row * a.ld_out;
    const float inv_f = 1.0f / (float)a.features;

    nh_raw<T, V> r[NV];
    float s = 0.0f, unused = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t c = (uint32_t)(k * TPR + t) * V;
        load_clipped(r[k], x + c, clip((long long)a.features - c, V));
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) s += r[k].get(j);
    row_sum2<TPR>(s, unused, slots[0]);
    const float mu = s * inv_f;
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int n = clip((long long)a.features - (uint32_t)(k * TPR + t) * V, V);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = r[k].get(j) - mu;
            q = __builtin_fmaf(d, j < n ? d : 0.0f, q);
        }
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
        const int n = clip((long long)a.features - c, V);
        if (n <= 0) continue;
        float g[V], b[V];
        load_floats<V>(g, a.gamma + c, n);
        load_floats<V>(b, a.beta + c, n);
        nh_out<T, V> o;
        o.clear();
#pragma unroll
        for (int j = 0; j < V; ++j) o.set(j, __builtin_fmaf((r[k].get(j) - mu) * rs, g[j], b[j]));
        store_clipped(o, y + c, n);
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
// ln_param_kernel adds up in a fixed order.
// ---------------------------------------------------------------------------
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void ln_rows_bprop_kernel(LnArgs a) {
    constexpr int V = vec<T>::V;
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float2 slots[2][TPR / 64];
    const int t = threadIdx.x % TPR;
    const float inv_f = 1.0f / (float)a.features;
    float g[NV][V], dg[NV][V], db[NV][V];
    int n[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t c = (uint32_t)(k * TPR + t) * V;
        n[k] = clip((long long)a.features - c, V);
        load_floats<V>(g[k], a.gamma + c, n[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) dg[k][j] = db[k][j] = 0.0f;
    }
    int parity = 0;
    const size_t step = (size_t)gridDim.x * RPB;
    for (size_t row = (size_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.positions; row += step) {
        const T* x = (const T*)a.x + row * a.ld_x;
        const T* dy = (const T*)a.dy + row * a.ld_dy;
        T* dx = (T*)a.out + row * a.ld_out;
        nh_raw<T, V> rx[NV], rd[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t c = (uint32_t)(k * TPR + t) * V;
            load_clipped(rx[k], x + c, n[k]);
            load_clipped(rd[k], dy + c, n[k]);
        }
        const float mu = a.mean[row], rs = inv_std(a.var[row], a.eps);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (rx[k].get(j) - mu) * rs, d = rd[k].get(j), u = d * g[k][j];
                s1 += u;
                s2 = __builtin_fmaf(u, h, s2);
                dg[k][j] = __builtin_fmaf(d, h, dg[k][j]);
                db[k][j] += d;
            }
        row_sum2<TPR>(s1, s2, slots[parity]);
        parity ^= 1;
        s1 *= inv_f;
        s2 *= inv_f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (n[k] <= 0) continue;
            nh_out<T, V> o;
            o.clear();
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (rx[k].get(j) - mu) * rs, u = rd[k].get(j) * g[k][j];
                o.set(j, rs * ((u - s1) - h * s2));
            }
            store_clipped(o, dx + (uint32_t)(k * TPR + t) * V, n[k]);
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
// strips of features in a kernel of their own
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

// grads[which][f] = sum of `count` partial rows, in a fixed order: 16 threads
// per feature take every 16th row, joined in LDS
__global__ __launch_bounds__(1024) void ln_param_kernel(LnArgs a, uint32_t count) {
    __shared__ float join[16][64];
    const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    const size_t f = (size_t)blockIdx.x * 64 + lane;
    const float* p = a.part + (size_t)blockIdx.y * a.features + f;
    float s = 0.0f;
    if (f < a.features)
        for (uint32_t i = grp; i < count; i += 16) s += p[(size_t)i * 2 * a.features];
    join[grp][lane] = s;
    __syncthreads();
    if (grp == 0 && f < a.features) {
#pragma unroll
        for (int w = 1; w < 16; ++w) s += join[w][lane];
        a.grads[blockIdx.y][f] = s;
    }
}

// ---------------------------------------------------------------------------
// columns: a workgroup takes a strip of 128 bytes of positions (8 lanes of 16
// bytes) and NT/8 x RV features at a time.  MODE 0: the strip's features fit
// one tile, which stays in registers (one read).  MODE 1 leaves the column
// sums of a run of tiles (blockIdx.y) in the workspace; MODE 2 joins them in
// order and finishes the same run.
// ---------------------------------------------------------------------------
constexpr int LC = 8;                 // lanes across a strip
enum { WHOLE = 0, SUMS = 1, FINISH = 2 };

template <typename T> struct strip { static constexpr int COLS = LC * vec<T>::V; };

// running (count, mean, sum of squared deviations) of two disjoint sets of a column's
// values joined: with the counts the same for all columns a thread holds, the two factors
// are computed once
struct JoinFactors {
    float to_b, cross;      // n_b / n and n_a n_b / n
    NEON_DEV JoinFactors(float na, float nb) {
        const float n = na + nb;
        to_b = n > 0.0f ? nb / n : 0.0f;
        cross = na * to_b;
    }
    NEON_DEV void join(float& mean, float& m2, float mean_b, float m2_b) const {
        const float d = mean_b - mean;
        mean = __builtin_fmaf(d, to_b, mean);
        m2 = (m2 + m2_b) + (d * d) * cross;
    }
};

template <typename T, int NT, int RV, int MODE>
__global__ __launch_bounds__(NT) void ln_cols_fprop_kernel(LnArgs a, uint32_t rows_per, uint32_t chunks) {
    constexpr int V = vec<T>::V, COLS = strip<T>::COLS, NW = NT / 64, RL = NT / LC;
    __shared__ float s_mean[NW][COLS], s_m2[NW][COLS], s_n[NW];
    const int t = threadIdx.x, cl = t % LC, rl = t / LC, wave = t >> 6;
    const size_t c0 = (size_t)blockIdx.x * COLS, c = c0 + cl * V;
    const int n = clip((long long)a.positions - (long long)c, V);
    const uint32_t r0 = MODE == WHOLE ? 0 : blockIdx.y * rows_per;
    const uint32_t r1 = MODE == WHOLE ? a.features : (r0 + rows_per < a.features ? r0 + rows_per : a.features);
    const T* x = (const T*)a.x + c;
    nh_raw<T, V> r[RV];
    float mean[V], m2[V];

    if constexpr (MODE != FINISH) {
#pragma unroll
        for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.0f;
        float cnt = 0.0f;
        for (uint32_t base = r0; base < r1; base += RL * RV) {
            int rows = 0;
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + rl + i * RL;
                if (f < r1) {
                    load_clipped(r[i], x + (size_t)f * a.ld_x, n);
                    ++rows;
                } else {
                    r[i].zero();
                }
            }
            const JoinFactors jf(cnt, (float)rows);
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
                jf.join(mean[j], m2[j], m, q);
            }
            cnt += (float)rows;
            if (MODE == WHOLE) break;
        }
        // lanes of a wave that share columns, then the waves
        {
            const auto fold = [&](auto S) {
                constexpr int X = decltype(S)::value;
                const float nb = nh_lane_xor<X>(cnt);
                const bool up = (t & X) != 0;
                // both partners join in the same order, so that they agree to the bit
                const JoinFactors jf(up ? nb : cnt, up ? cnt : nb);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float om = nh_lane_xor<X>(mean[j]), oq = nh_lane_xor<X>(m2[j]);
                    float ma = up ? om : mean[j], qa = up ? oq : m2[j];
                    jf.join(ma, qa, up ? mean[j] : om, up ? m2[j] : oq);
                    mean[j] = ma;
                    m2[j] = qa;
                }
                cnt += nb;
            };
            fold(std::integral_constant<int, 8>());
            fold(std::integral_constant<int, 16>());
            fold(std::integral_constant<int, 32>());
        }
        if ((t & 63) < LC) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s_mean[wave][cl * V + j] = mean[j];
                s_m2[wave][cl * V + j] = m2[j];
            }
            if (cl == 0) s_n[wave] = cnt;
        }
        __syncthreads();
        if (t < COLS) {
            float m = s_mean[0][t], q = s_m2[0][t], k = s_n[0];
            for (int w = 1; w < NW; ++w) {
                JoinFactors(k, s_n[w]).join(m, q, s_mean[w][t], s_m2[w][t]);
                k += s_n[w];
            }
            if (MODE == SUMS) {
                float* p = a.part + (((size_t)blockIdx.x * chunks + blockIdx.y) * COLS + t) * 2;
                p[0] = m;
                p[1] = q;
            } else {
                s_mean[0][t] = m;
                s_m2[0][t] = q;
            }
        }
    } else {
        if (t < COLS) {
            float m = 0.0f, q = 0.0f, k = 0.0f;
            for (uint32_t i = 0; i < chunks; ++i) {
                const float* p = a.part + (((size_t)blockIdx.x * chunks + i) * COLS + t) * 2;
                const uint32_t b = i * rows_per, e = b + rows_per < a.features ? b + rows_per : a.features;
                JoinFactors(k, (float)(e - b)).join(m, q, p[0], p[1]);
                k += (float)(e - b);
            }
            s_mean[0][t] = m;
            s_m2[0][t] = q;
        }
    }
    if constexpr (MODE != SUMS) {
        __syncthreads();
        const float inv_f = 1.0f / (float)a.features;
        if (t < COLS && c0 + t < a.positions && (MODE == WHOLE || blockIdx.y == 0)) {
            a.mean[c0 + t] = s_mean[0][t];
            a.var[c0 + t] = s_m2[0][t] * inv_f;
        }
        if (n <= 0) return;
        float rs[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            mean[j] = s_mean[0][cl * V + j];
            rs[j] = inv_std(s_m2[0][cl * V + j] * inv_f, a.eps);
        }
        T* y = (T*)a.out + c;
        for (uint32_t base = r0; base < r1; base += RL * RV) {
            if constexpr (MODE == FINISH) {
#pragma unroll
                for (int i = 0; i < RV; ++i) {
                    const uint32_t f = base + rl + i * RL;
                    if (f < r1) load_clipped(r[i], x + (size_t)f * a.ld_x, n);
                }
            }
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + rl + i * RL;
                if (f >= r1) continue;
                const float g = a.gamma[f], b = a.beta[f];
                nh_out<T, V> o;
                o.clear();
#pragma unroll
                for (int j = 0; j < V; ++j) o.set(j, __builtin_fmaf((r[i].get(j) - mean[j]) * rs[j], g, b));
                store_clipped(o, y + (size_t)f * a.ld_out, n);
            }
            if (MODE == WHOLE) break;
        }
    }
}

template <typename T, int NT, int RV, int MODE>
__global__ __launch_bounds__(NT) void ln_cols_bprop_kernel(LnArgs a, uint32_t rows_per, uint32_t chunks, float* sums) {
    constexpr int V = vec<T>::V, COLS = strip<T>::COLS, NW = NT / 64, RL = NT / LC;
    __shared__ float s_a[NW][COLS], s_b[NW][COLS];
    const int t = threadIdx.x, cl = t % LC, rl = t / LC, wave = t >> 6;
    const size_t c0 = (size_t)blockIdx.x * COLS, c = c0 + cl * V;
    const int n = clip((long long)a.positions - (long long)c, V);
    const uint32_t r0 = MODE == WHOLE ? 0 : blockIdx.y * rows_per;
    const uint32_t r1 = MODE == WHOLE ? a.features : (r0 + rows_per < a.features ? r0 + rows_per : a.features);
    const T* x = (const T*)a.x + c;
    const T* dy = (const T*)a.dy + c;
    nh_raw<T, V> rx[RV], rd[RV];
    float mu[V], rs[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        mu[j] = j < n ? a.mean[c + j] : 0.0f;
        rs[j] = j < n ? inv_std(a.var[c + j], a.eps) : 0.0f;
    }
    if constexpr (MODE != FINISH) {
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
        float* part = a.part + (size_t)blockIdx.x * 2 * a.features;
        for (uint32_t base = r0; base < r1; base += RL * RV) {
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + rl + i * RL;
                const int m = f < r1 ? n : 0;
                load_clipped(rx[i], x + (size_t)f * a.ld_x, m);
                load_clipped(rd[i], dy + (size_t)f * a.ld_dy, m);
            }
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + rl + i * RL;
                const float g = f < r1 ? a.gamma[f] : 0.0f;
                float dg = 0.0f, db = 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float h = (rx[i].get(j) - mu[j]) * rs[j], d = rd[i].get(j), u = d * g;
                    s1[j] += u;
                    s2[j] = __builtin_fmaf(u, h, s2[j]);
                    dg = __builtin_fmaf(d, h, dg);
                    db += d;
                }
                dg = nh_wave_allreduce<nh_op_sum, LC>(dg);
                db = nh_wave_allreduce<nh_op_sum, LC>(db);
                if (cl == 0 && f < r1) {
                    part[f] = dg;
                    part[a.features + f] = db;
                }
            }
            if (MODE == WHOLE) break;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s1[j] += nh_lane_xor<8>(s1[j]);
            s2[j] += nh_lane_xor<8>(s2[j]);
            s1[j] += nh_lane_xor<16>(s1[j]);
            s2[j] += nh_lane_xor<16>(s2[j]);
            s1[j] += nh_lane_xor<32>(s1[j]);
            s2[j] += nh_lane_xor<32>(s2[j]);
        }
        if ((t & 63) < LC) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s_a[wave][cl * V + j] = s1[j];
                s_b[wave][cl * V + j] = s2[j];
            }
        }
        __syncthreads();
        if (t < COLS) {
            float p = s_a[0][t], q = s_b[0][t];
            for (int w = 1; w < NW; ++w) {
                p += s_a[w][t];
                q += s_b[w][t];
            }
            if (MODE == SUMS) {
                float* o = sums + (((size_t)blockIdx.x * chunks + blockIdx.y) * COLS + t) * 2;
                o[0] = p;
                o[1] = q;
            } else {
                s_a[0][t] = p;
                s_b[0][t] = q;
            }
        }
    } else {
        if (t < COLS) {
            float p = 0.0f, q = 0.0f;
            for (uint32_t i = 0; i < chunks; ++i) {
                const float* o = sums + (((size_t)blockIdx.x * chunks + i) * COLS + t) * 2;
                p += o[0];
                q += o[1];
            }
            s_a[0][t] = p;
            s_b[0][t] = q;
        }
    }
    if constexpr (MODE != SUMS) {
        __syncthreads();
        if (n <= 0) return;
        const float inv_f = 1.0f / (float)a.features;
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s1[j] = s_a[0][cl * V + j] * inv_f;
            s2[j] = s_b[0][cl * V + j] * inv_f;
        }
        T* dx = (T*)a.out + c;
        for (uint32_t base = r0; base < r1; base += RL * RV) {
            if constexpr (MODE == FINISH) {
#pragma unroll
                for (int i = 0; i < RV; ++i) {
                    const uint32_t f = base + rl + i * RL;
                    const int m = f < r1 ? n : 0;
                    load_clipped(rx[i], x + (size_t)f * a.ld_x, m);
                    load_clipped(rd[i], dy + (size_t)f * a.ld_dy, m);
                }
            }
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const uint32_t f = base + rl + i * RL;
                if (f >= r1) continue;
                const float g = a.gamma[f];
                nh_out<T, V> o;
                o.clear();
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float h = (rx[i].get(j) - mu[j]) * rs[j], u = rd[i].get(j) * g;
                    o.set(j, rs[j] * ((u - s1[j]) - h * s2[j]));
                }
                store_clipped(o, dx + (size_t)f * a.ld_out, n);
            }
            if (MODE == WHOLE) break;
        }
    }
}

// ---------------------------------------------------------------------------
// launch geometry
// ---------------------------------------------------------------------------
constexpr size_t LONG_ROW_FPROP = 65536;      // features one workgroup's registers hold
constexpr size_t LONG_ROW_BPROP = 16384;
constexpr unsigned ROW_GROUPS = 512;          // workgroups that walk the rows in the backward pass
constexpr unsigned LONG_ROW_RUNS = 64;        // row runs per feature strip in ln_rows_params_kernel
constexpr size_t COL_TILE = 256;              // features per tile of the split column kernels
constexpr size_t COL_RESIDENT = 1024;         // features a 1024-thread workgroup keeps
constexpr size_t COL_CHUNKS = 32;             // runs of tiles per strip, at most

size_t strip_cols(int dtype) { return (size_t)128 / lm::item_bytes(dtype); }

struct ColSplit {
    uint32_t rows_per, chunks;
};
ColSplit split_columns(size_t features) {
    const size_t tiles = lm::ceil_div(features, COL_TILE);
    const size_t per = lm::ceil_div(tiles, COL_CHUNKS);
    return {(uint32_t)(per * COL_TILE), (uint32_t)lm::ceil_div(tiles, per)};
}

unsigned row_groups(size_t features, size_t positions, int dtype) {
    const size_t per_block = features <= (size_t)64 * 16 ? 4 : 1;
    const size_t blocks = lm::ceil_div(positions, per_block);
    return (unsigned)(blocks < ROW_GROUPS ? blocks : ROW_GROUPS);
}

size_t partial_rows(size_t features, size_t positions, int dtype, bool columns) {
    if (columns) return lm::ceil_div(positions, strip_cols(dtype));
    if (features > LONG_ROW_BPROP) return positions < LONG_ROW_RUNS ? positions : LONG_ROW_RUNS;
    return row_groups(features, positions, dtype);
}

size_t column_sum_bytes(size_t features, size_t positions, int dtype) {
    return lm::align256(lm::ceil_div(positions, strip_cols(dtype)) * split_columns(features).chunks * strip_cols(dtype) * 2 *
                        sizeof(float));
}

size_t workspace_bytes(bool backward, int dtype, bool columns, size_t features, size_t positions) {
    size_t need = 0;
    if (columns && features > COL_RESIDENT) need += column_sum_bytes(features, positions, dtype);
    if (backward) need += lm::align256(partial_rows(features, positions, dtype, columns) * 2 * features * sizeof(float));
    return need;
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

template <typename T> int fprop_rows(const LnArgs& a, hipStream_t s) {
    constexpr size_t V = vec<T>::V;
    const size_t nvec = lm::ceil_div(a.features, V);
    if (a.positions > lm::MAX_BLOCKS) return lm::refuse("nh_ln_fprop", "too many positions for one launch");
    const dim3 by4((unsigned)lm::ceil_div(a.positions, 4)), by1((unsigned)a.positions);
#define LN_GO(TPR, NV) hipLaunchKernelGGL((ln_rows_fprop_kernel<T, TPR, NV>), TPR == 64 ? by4 : by1, dim3(TPR == 64 ? 256 : TPR), 0, s, a)
    if (nvec <= 64) LN_GO(64, 1);
    else if (nvec <= 128) LN_GO(64, 2);
    else if (nvec <= 256) LN_GO(256, 1);
    else if (nvec <= 512) LN_GO(256, 2);
    else if (nvec <= 1024) LN_GO(256, 4);
    else if (nvec <= 2048) LN_GO(1024, 2);
    else if (nvec <= 4096) LN_GO(1024, 4);
    else if (nvec <= 8192) LN_GO(1024, 8);
    else if (a.features > LONG_ROW_FPROP) hipLaunchKernelGGL((ln_rows_fprop_long_kernel<T>), by1, dim3(1024), 0, s, a);
    else if constexpr (sizeof(T) == 4) LN_GO(1024, 16);
#undef LN_GO
    return lm::launched("nh_ln_fprop");
}

template <typename T> int fprop_cols(const LnArgs& a, hipStream_t s) {
    const size_t strips = lm::ceil_div(a.positions, strip<T>::COLS);
    if (strips > lm::MAX_BLOCKS) return lm::refuse("nh_ln_fprop", "too many positions for one launch");
    if (a.features <= COL_TILE) {
        hipLaunchKernelGGL((ln_cols_fprop_kernel<T, 256, 8, WHOLE>), dim3((unsigned)strips), dim3(256), 0, s, a, 0u, 1u);
    } else if (a.features <= COL_RESIDENT) {
        hipLaunchKernelGGL((ln_cols_fprop_kernel<T, 1024, 8, WHOLE>), dim3((unsigned)strips), dim3(1024), 0, s, a, 0u, 1u);
    } else {
        const ColSplit c = split_columns(a.features);
        const dim3 grid((unsigned)strips, c.chunks);
        hipLaunchKernelGGL((ln_cols_fprop_kernel<T, 256, 8, SUMS>), grid, dim3(256), 0, s, a, c.rows_per, c.chunks);
        hipLaunchKernelGGL((ln_cols_fprop_kernel<T, 256, 8, FINISH>), grid, dim3(256), 0, s, a, c.rows_per, c.chunks);
    }
    return lm::launched("nh_ln_fprop");
}

void add_params(const LnArgs& a, size_t count, hipStream_t s) {
    hipLaunchKernelGGL(ln_param_kernel, dim3((unsigned)lm::ceil_div(a.features, 64), 2), dim3(1024), 0, s, a, (uint32_t)count);
}

template <typename T> int bprop_rows(const LnArgs& a, hipStream_t s) {
    constexpr size_t V = vec<T>::V;
    const size_t nvec = lm::ceil_div(a.features, V);
    const size_t rows = partial_rows(a.features, a.positions, sizeof(T) == 4 ? NH_T_F32 : NH_T_F16, false);
    if (a.features > LONG_ROW_BPROP) {
        if (a.positions > lm::MAX_BLOCKS) return lm::refuse("nh_ln_bprop", "too many positions for one launch");
        const size_t per = lm::ceil_div(a.positions, rows);
        // (the sums first: dx may take the place of dy)
        hipLaunchKernelGGL((ln_rows_params_kernel<T>), dim3((unsigned)lm::ceil_div(nvec, 64), (unsigned)rows), dim3(64), 0, s, a, per);
        hipLaunchKernelGGL((ln_rows_bprop_long_kernel<T>), dim3((unsigned)a.positions), dim3(1024), 0, s, a);
        add_params(a, rows, s);
        return lm::launched("nh_ln_bprop");
    }
    const dim3 grid((unsigned)rows);
#define LN_GO(TPR, NV) hipLaunchKernelGGL((ln_rows_bprop_kernel<T, TPR, NV>), grid, dim3(TPR == 64 ? 256 : TPR), 0, s, a)
    if (a.features <= 64 * V) LN_GO(64, 1);
    else if (a.features <= 64 * 8) LN_GO(64, 8 / V < 2 ? 1 : 2);
    else if (a.features <= 64 * 16) LN_GO(64, 16 / V);
    else if (a.features <= 256 * 8) LN_GO(256, 8 / V);
    else if (a.features <= 256 * 16) LN_GO(256, 16 / V);
    else if (a.features <= 1024 * 8) LN_GO(1024, 8 / V);
    else LN_GO(1024, 16 / V);
#undef LN_GO
    add_params(a, rows, s);
    return lm::launched("nh_ln_bprop");
}

template <typename T> int bprop_cols(LnArgs a, char* ws, hipStream_t s) {
    const size_t strips = lm::ceil_div(a.positions, strip<T>::COLS);
    if (strips > lm::MAX_BLOCKS) return lm::refuse("nh_ln_bprop", "too many positions for one launch");
    if (a.features <= COL_TILE) {
        a.part = (float*)ws;
        hipLaunchKernelGGL((ln_cols_bprop_kernel<T, 256, 8, WHOLE>), dim3((unsigned)strips), dim3(256), 0, s, a, 0u, 1u, nullptr);
    } else if (a.features <= COL_RESIDENT) {
        a.part = (float*)ws;
        hipLaunchKernelGGL((ln_cols_bprop_kernel<T, 1024, 8, WHOLE>), dim3((unsigned)strips), dim3(1024), 0, s, a, 0u, 1u, nullptr);
    } else {
        const ColSplit c = split_columns(a.features);
        const dim3 grid((unsigned)strips, c.chunks);
        float* sums = (float*)ws;
        a.part = (float*)(ws + column_sum_bytes(a.features, a.positions, sizeof(T) == 4 ? NH_T_F32 : NH_T_F16));
        hipLaunchKernelGGL((ln_cols_bprop_kernel<T, 256, 8, SUMS>), grid, dim3(256), 0, s, a, c.rows_per, c.chunks, sums);
        hipLaunchKernelGGL((ln_cols_bprop_kernel<T, 256, 8, FINISH>), grid, dim3(256), 0, s, a, c.rows_per, c.chunks, sums);
    }
    add_params(a, strips, s);
    return lm::launched("nh_ln_bprop");
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
    if (!nh_internal_ready()) return nh_internal_fail(NH_ENOTINIT, "nh_init has not been called");
    lm::OnDevice here;
    LnArgs a = {};
    a.x = x; a.out = y; a.gamma = gamma; a.beta = beta; a.mean = mean; a.var = var; a.part = (float*)workspace;
    a.eps = eps; a.features = (uint32_t)features; a.positions = positions; a.ld_x = ld_x; a.ld_out = ld_y;
    return lm::by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return axis == 1 ? fprop_rows<T>(a, (hipStream_t)stream) : fprop_cols<T>(a, (hipStream_t)stream);
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
    if (!nh_internal_ready()) return nh_internal_fail(NH_ENOTINIT, "nh_init has not been called");
    lm::OnDevice here;
    LnArgs a = {};
    a.x = x; a.dy = dy; a.out = dx; a.gamma = gamma; a.mean = const_cast<float*>(mean); a.var = const_cast<float*>(var);
    a.part = (float*)workspace; a.grads[0] = dgamma; a.grads[1] = dbeta;
    a.eps = eps; a.features = (uint32_t)features; a.positions = positions; a.ld_x = ld_x; a.ld_dy = ld_dy; a.ld_out = ld_dx;
    if (positions == 0) {          // sums over no positions
        add_params(a, 0, (hipStream_t)stream);
        return lm::launched("nh_ln_bprop");
    }
    return lm::by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return axis == 1 ? bprop_rows<T>(a, (hipStream_t)stream) : bprop_cols<T>(a, (char*)workspace, (hipStream_t)stream);
    });
}

}  // extern "C"
