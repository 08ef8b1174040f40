// GroupNorm + scale/shift + activation + residual of a channels-last tensor (any group count), and its backward (gfx950).
//   u = gamma' (x - mean) rstd + beta',  gamma' = gamma (1 + scale_b),  beta' = beta (1 + scale_b) + shift_b,  y = act(u) [+ res]
// with mean / rstd per (image, group); the adjoint in terms of the forward's (mean, rstd):
//   du = dy act'(u),  S1[b,c] = sum_p du,  S2[b,c] = sum_p du xhat,  m1 / m2 = group means of gamma' du / gamma' du xhat,
//   dx = rstd (gamma' du - m1 - xhat m2),  dgamma = sum_b (1 + scale) S2,  dbeta = sum_b (1 + scale) S1,
//   dscale = gamma S2 + beta S1,  dshift = S1.
// Everything between the loads and the stores is fp32, sums across threads fp64, and a thread's own sums where they are long (LONG); a block's or a split's
// sums are stored in fp32.  The only rounding to bf16 is the stored result.
// No atomics: partial sums lie in the workspace and are added in a fixed order, and how an image is split depends on its own
// size only, so a result does not depend on the batch it is computed in - but for the backward of larger images, many of
// which go to one block each while few are split (bwd_one_block).
#include <type_traits>

#include "act.hpp"

namespace {

constexpr int NT = 256;
// Rows that a thread adds in fp32.  Where it has more than ROWS_MAX of them, it closes its sums every CHAIN rows and goes on in fp64 (LONG), in its own
// place in LDS, so that the error does not grow with the image.  Not so below: the closing costs loads in flight (1x65536x512 bf16, 256 rows a thread: 55 us
// unclosed, 69 closed, 50 closed over twice as many splits, see geo_of; 32x65536x64, 32 rows: 142 against 146).
constexpr int ROWS_MAX = 64, CHAIN = 32;

// V consecutive channels of one row as they lie in memory (V = 8: 16-byte aligned vectors; V = 1: any alignment)
template <typename T, int V> struct Raw;
template <typename T> struct Raw<T, 8> {
    Frag<T> f;
    __device__ __forceinline__ void load(const T* p) { frag_load<T>(f, p); }
    __device__ __forceinline__ void load_once(const T* p) {  // its lines are not kept in the caches
        f32x4 q[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) q[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p) + i);
        __builtin_memcpy(&f, q, sizeof(f));
    }
    __device__ __forceinline__ float get(int j) const { return frag_get<T>(f, j); }
};
template <typename T> struct Raw<T, 1> {
    T f;
    __device__ __forceinline__ void load(const T* p) { f = *p; }
    __device__ __forceinline__ void load_once(const T* p) { f = *p; }
    __device__ __forceinline__ float get(int) const { return to_f32<T>(f); }
};
template <typename T, int V> __device__ __forceinline__ void vstore(const float (&f)[V], T* p) {
    if constexpr (V == 8) {
        Frag<T> q;
#pragma unroll
        for (int j = 0; j < 8; j++) frag_set<T>(q, j, f[j]);
        frag_store<T>(q, p);
    } else {
        *p = from_f32<T>(f[0]);
    }
}
template <typename T, int V> __device__ __forceinline__ void vstore_once(const float (&f)[V], T* p) {
    if constexpr (V == 8) {
        Frag<T> g;
#pragma unroll
        for (int j = 0; j < 8; j++) frag_set<T>(g, j, f[j]);
        f32x4 q[sizeof(T) / 2];
        __builtin_memcpy(q, &g, sizeof(g));
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) __builtin_nontemporal_store(q[i], reinterpret_cast<f32x4*>(p) + i);
    } else {
        *p = from_f32<T>(f[0]);
    }
}
// a thread's n rows, `step` elements apart, U of them in flight: body(vector, row number).  ONCE: the last use of what is read
template <int U, typename T, int V, bool ONCE = false, typename F> __device__ __forceinline__ void each_row(const T* p, size_t step, int n, F&& body) {
    int i = 0;
    for (; i + U <= n; i += U, p += U * step) {
        Raw<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; u++) ONCE ? v[u].load_once(p + u * step) : v[u].load(p + u * step);
#pragma unroll
        for (int u = 0; u < U; u++) body(v[u], i + u);
    }
    if (i < n) {
        Raw<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u < n) ONCE ? v[u].load_once(p + u * step) : v[u].load(p + u * step);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u < n) body(v[u], i + u);
    }
}
template <int U, typename T, int V, bool ONCE = false, typename F>
__device__ __forceinline__ void each_row2(const T* p, size_t pstep, const T* d, size_t dstep, int n, F&& body) {
    int i = 0;
    for (; i + U <= n; i += U, p += U * pstep, d += U * dstep) {
        Raw<T, V> v[U], w[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            ONCE ? v[u].load_once(p + u * pstep) : v[u].load(p + u * pstep);
            ONCE ? w[u].load_once(d + u * dstep) : w[u].load(d + u * dstep);
        }
#pragma unroll
        for (int u = 0; u < U; u++) body(v[u], w[u], i + u);
    }
    if (i < n) {
        Raw<T, V> v[U], w[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u < n) {
                ONCE ? v[u].load_once(p + u * pstep) : v[u].load(p + u * pstep);
                ONCE ? w[u].load_once(d + u * dstep) : w[u].load(d + u * dstep);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u < n) body(v[u], w[u], i + u);
    }
}

// How an image is cut: chunks of channels (LP lanes x V channels), R rows at a time in a block, S splits of RS rows: as many as leave a thread 8 rows, at
// most 64, or 128 of images where a thread would have more than ROWS_MAX rows.  More splits cost their joins: 128 for 32x65536x64 bf16, 32 rows a thread in
// 64, 156 us against 146; for 1x65536x512, 256 rows, they are ahead, 50 against 69 forward and 79 against 163 backward.
struct Geo {
    int P, C, G, cg, LP, R, CH, nch, S, RS;
};

__host__ __device__ inline Geo geo_of(int P, int C, int G, int V, int rows_per_thread) {
    Geo q;
    q.P = P;
    q.C = C;
    q.G = G;
    q.cg = C / G;
    const int vecs = (C + V - 1) / V;
    q.LP = vecs < NT ? vecs : NT;
    q.R = NT / q.LP;
    q.CH = q.LP * V;
    q.nch = (C + q.CH - 1) / q.CH;
    int S = (P + q.R * rows_per_thread - 1) / (q.R * rows_per_thread);
    const int most = P > 64 * ROWS_MAX * q.R ? 128 : 64;
    if (S > most) S = most;
    if (S < 1) S = 1;
    q.RS = (P + S - 1) / S;
    q.S = (P + q.RS - 1) / q.RS;
    return q;
}

__device__ __forceinline__ int rows_of(int P, int ty, int R) { return P > ty ? (P - ty + R - 1) / R : 0; }

struct FwdP {
    const void* x;
    const float *gamma, *beta, *ss;
    const void* res;
    void* out;
    float *mr, *part;
    long long x_bs, x_ld, r_bs, r_ld;
    int ss_ld, ss_off, wide;  // wide: gamma, beta and ss can be read 16 bytes at a time
    float eps;
    Geo q;
};

// ---- pass 1: (mean, M2) of every (image, group, split): per-thread sums about the thread's own first sample.  A sum of n squares about one of the
// samples is at most n + 1 times their M2, so the subtraction S2 - S1^2 / n loses at most about n ulps, whatever the mean; n is at most ROWS_MAX.
// LONG: runs of CHAIN rows, about the mean of the first 8 rows and later of all rows before the run.  With k rows behind the pivot, S2 of a run of n is at most
// 1 + n / k (the first run) or 2 + n / k times the M2 of all these rows: 5 in the first run, 3 in the second, then less; runs are joined as (mean, M2) in fp64.
// Bound by HBM: 32x65536x64 bf16 55 us = 4.9 TB/s.
template <typename T, int V, bool LONG> __global__ __launch_bounds__(NT) void gn_stats_kernel(FwdP p) {
    using Sum = std::conditional_t<LONG, double, float>;
    __shared__ Sum sm_mean[NT * V], sm_m2[NT * V];
    const Geo q = p.q;
    int id = blockIdx.x;
    const int s = id % q.S;
    id /= q.S;
    const int ch = id % q.nch, b = id / q.nch;
    const int tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int c0 = ch * q.CH, c = c0 + tx * V;
    const int row0 = s * q.R, cycle = q.S * q.R;  // R rows at a time, dealt round over the splits
    const bool on = ty < q.R && c < q.C;
    if (on) {
        const int n = rows_of(q.P, row0 + ty, cycle);
        const T* x = (const T*)p.x + (size_t)b * p.x_bs + (size_t)(row0 + ty) * p.x_ld + c;
        const size_t step = (size_t)cycle * p.x_ld;
        Sum *mean = sm_mean + ty * q.CH + tx * V, *m2 = sm_m2 + ty * q.CH + tx * V;
        float piv[V], s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; j++) piv[j] = 0.f;
        auto run = [&](int rows) {
#pragma unroll
            for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
            each_row<8, T, V>(x, step, rows, [&](const Raw<T, V>& v, int i) {
                if (!LONG && i == 0) {
#pragma unroll
                    for (int j = 0; j < V; j++) piv[j] = v.get(j);
                }
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = v.get(j) - piv[j];
                    s1[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
            });
            const float inv = rows > 0 ? 1.f / (float)rows : 0.f;
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float m = s1[j] * inv;
                s2[j] -= s1[j] * m;
                s1[j] = piv[j] + m;
            }
        };
        if constexpr (LONG) {  // n >= ROWS_MAX
            Raw<T, V> v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u].load(x + u * step);
#pragma unroll
            for (int j = 0; j < V; j++) {
                float t = 0.f;
#pragma unroll
                for (int u = 1; u < 8; u++) t += v[u].get(j) - v[0].get(j);
                piv[j] = fmaf(t, 0.125f, v[0].get(j));
            }
            for (int done = 0; done < n;) {
                const int rows = min(CHAIN, n - done);
                run(rows);
                x += rows * step;
                const double w = (double)rows / (double)(done + rows), wd = w * (double)done;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const double was = done ? mean[j] : 0.0, d = (double)s1[j] - was;
                    mean[j] = was + d * w;
                    m2[j] = (done ? m2[j] : 0.0) + (double)s2[j] + d * d * wd;
                    piv[j] = (float)mean[j];
                }
                done += rows;
            }
        } else {
            run(n);
#pragma unroll
            for (int j = 0; j < V; j++) {
                mean[j] = s1[j];
                m2[j] = s2[j];
            }
        }
    }
    __syncthreads();
    // groups that meet this chunk: weighted mean, then M2 about it.  A wave takes one, or all four share it where there is only one;
    // a row y of the block stands for `base` rows of the image, or one more.
    __shared__ double sm_w[NT / 64][2];
    const int c1 = min(q.C, c0 + q.CH), g0 = c0 / q.cg, g1 = (c1 - 1) / q.cg, lane = tid & 63, wave = tid >> 6;
    const int base = q.P / cycle, extra = q.P - base * cycle - row0;
    const bool shared = g0 == g1;
    for (int g = g0 + (shared ? 0 : wave); g <= g1; g += NT / 64) {
        const int lo = max(c0, g * q.cg) - c0, hi = min(c1, (g + 1) * q.cg) - c0, w = hi - lo;
        // lanes x channels x rows without a division in the loop: narrow groups put 64 / w rows side by side
        const int side = w < 64 ? 64 / w : 1, y0 = w < 64 ? lane / w : 0, e0 = w < 64 ? lane - y0 * w : lane, per = shared ? NT / 64 : 1;
        const int yfirst = y0 + (shared ? wave * side : 0), ystep = side * per;
        const bool in = y0 < side;
        double sn = 0.0, sm = 0.0;
        if (in)
            for (int y = yfirst; y < q.R; y += ystep) {
                const double n = (double)(base + (y < extra ? 1 : 0));
                for (int e = e0; e < w; e += 64) {
                    sm += n > 0.0 ? n * (double)sm_mean[y * q.CH + lo + e] : 0.0;
                    sn += n;
                }
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            sm += __shfl_xor(sm, o, 64);
            sn += __shfl_xor(sn, o, 64);
        }
        if (shared) {  // the loop is left by all waves together
            if (lane == 0) {
                sm_w[wave][0] = sm;
                sm_w[wave][1] = sn;
            }
            __syncthreads();
            sm = (sm_w[0][0] + sm_w[1][0]) + (sm_w[2][0] + sm_w[3][0]);
            sn = (sm_w[0][1] + sm_w[1][1]) + (sm_w[2][1] + sm_w[3][1]);
            __syncthreads();
        }
        const double mean = sm / sn;
        double m2 = 0.0;
        if (in)
            for (int y = yfirst; y < q.R; y += ystep) {
                const double n = (double)(base + (y < extra ? 1 : 0));
                if (n > 0.0)
                    for (int e = e0; e < w; e += 64) {
                        const int i = y * q.CH + lo + e;
                        const double d = (double)sm_mean[i] - mean;
                        m2 += (double)sm_m2[i] + n * d * d;
                    }
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
        if (shared) {
            if (lane == 0) sm_w[wave][0] = m2;
            __syncthreads();
            m2 = (sm_w[0][0] + sm_w[1][0]) + (sm_w[2][0] + sm_w[3][0]);
        }
        if (lane == 0 && (!shared || wave == 0)) {
            float* d = p.part + (((size_t)b * q.G + g) * (q.nch * q.S) + ch * q.S + s) * 2;
            d[0] = (float)mean;
            d[1] = (float)m2;
        }
    }
}

// rows of split s times channels of group g in chunk ch
__device__ __forceinline__ double entry_count(const Geo& q, int g, int e) {
    const int ch = e / q.S, s = e - ch * q.S;
    const int cycle = q.S * q.R, rows = q.P / cycle * q.R + min(max(q.P % cycle - s * q.R, 0), q.R);
    const int w = min(min(q.C, (ch + 1) * q.CH), (g + 1) * q.cg) - max(ch * q.CH, g * q.cg);
    return w > 0 ? (double)rows * (double)w : 0.0;
}

// ---- pass 2: one wave per (image, group) joins the partials: mean, then M2 about it, in fp64
__device__ __forceinline__ void gn_join(const FwdP& p, int b, int g, int lane, float& mean_o, float& rstd_o) {
    const Geo& q = p.q;
    const int E = q.nch * q.S;
    const float* src = p.part + ((size_t)b * q.G + g) * E * 2;
    double sm = 0.0;
    for (int e = lane; e < E; e += 64) {
        const double n = entry_count(q, g, e);
        if (n > 0.0) sm += n * (double)src[2 * e];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sm += __shfl_xor(sm, o, 64);
    const double n_all = (double)q.P * (double)q.cg, mean = sm / n_all;
    double m2 = 0.0;
    for (int e = lane; e < E; e += 64) {
        const double n = entry_count(q, g, e);
        if (n > 0.0) {
            const double d = (double)src[2 * e] - mean;
            m2 += (double)src[2 * e + 1] + n * d * d;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
    mean_o = (float)mean;
    rstd_o = (float)(1.0 / sqrt(m2 / n_all + (double)p.eps));
}

__global__ __launch_bounds__(NT) void gn_join_kernel(FwdP p, long long n) {
    const long long i = (long long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    if (i >= n) return;
    const int b = (int)(i / p.q.G), g = (int)(i - (long long)b * p.q.G), lane = threadIdx.x & 63;
    float m, r;
    gn_join(p, b, g, lane, m, r);
    if (lane == 0) {
        p.mr[2 * i] = m;
        p.mr[2 * i + 1] = r;
    }
}

// gamma', beta' of one channel
__device__ __forceinline__ void affine_of(const float* gamma, const float* beta, const float* ss, int ss_ld, int ss_off, int b, int C, int c, float& a, float& o,
                                          float& sc) {
    a = gamma[c];
    o = beta[c];
    sc = 1.f;
    if (ss) {
        const float* row = ss + (size_t)b * ss_ld + ss_off;
        sc = 1.f + row[c];
        a *= sc;
        o = fmaf(o, sc, row[C + c]);
    }
}

// the same for V channels from c, and beta (1 + scale)
template <int V, typename P> __device__ __forceinline__ void affine_vec(const P& p, int b, int c, float (&a)[V], float (&o)[V], float (&bt)[V]) {
    float sc[V], sh[V];
    const float* row = p.ss ? p.ss + (size_t)b * p.ss_ld + p.ss_off + c : nullptr;
    if (V == 8 && p.wide) {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
            *reinterpret_cast<f32x4*>(a + h) = *reinterpret_cast<const f32x4*>(p.gamma + c + h);
            *reinterpret_cast<f32x4*>(bt + h) = *reinterpret_cast<const f32x4*>(p.beta + c + h);
            if (row) {
                *reinterpret_cast<f32x4*>(sc + h) = *reinterpret_cast<const f32x4*>(row + h);
                *reinterpret_cast<f32x4*>(sh + h) = *reinterpret_cast<const f32x4*>(row + p.q.C + h);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) {
            a[j] = p.gamma[c + j];
            bt[j] = p.beta[c + j];
            if (row) {
                sc[j] = row[j];
                sh[j] = row[p.q.C + j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (row) {
            const float f = 1.f + sc[j];
            a[j] *= f;
            o[j] = fmaf(bt[j], f, sh[j]);
            bt[j] *= f;
        } else {
            o[j] = bt[j];
        }
    }
}
// the pair [group of channel c + j][2] at `pairs` of V channels
template <int V> __device__ __forceinline__ void group_pairs(const float* pairs, int cg, int c, float (&x)[V], float (&y)[V]) {
    if (V == 8 && cg % 8 == 0) {  // c is a multiple of 8: one group
        const int g = c / cg;
        const float u = pairs[2 * g], v = pairs[2 * g + 1];
#pragma unroll
        for (int j = 0; j < V; j++) {
            x[j] = u;
            y[j] = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int g = (c + j) / cg;
            x[j] = pairs[2 * g];
            y[j] = pairs[2 * g + 1];
        }
    }
}

// Factors of u = mul (x - mean) + add for the channels of a thread.  The mean is taken off x first: folded into add (one instruction less) it would leave
// U |mean| mul of absolute error (U = 2^-24), and mul goes up to 316 gamma' where a group is constant - xhat is 0 there and u has to be beta'.
// SiLU's factors are scaled by -log2 e (silu_pre).
template <typename T, int V, int ACT> struct Affine {
    float mean[V], mul[V], add[V];
    __device__ __forceinline__ void set(int j, float m, float mu, float ad) {
        mean[j] = m;
        mul[j] = ACT == ACT_SILU ? mu * SILU_PRE : mu;
        add[j] = ACT == ACT_SILU ? ad * SILU_PRE : ad;
    }
    __device__ __forceinline__ float value(int j, float x) const {
        const float xc = x - mean[j];
        if constexpr (ACT == ACT_SILU) return silu_pre(mul[j], add[j], xc);
        else return act_val<T, ACT>(fmaf(xc, mul[j], add[j]));
    }
};

// ---- pass 3: y = act(gamma' (x - mean) rstd + beta') + res.  With few partials per image (JOIN_MAX) every block joins its groups
// itself and pass 2 is not launched.
constexpr int JOIN_GROUPS = 16, JOIN_MAX = 1024;
// Blocks run from the last image to the first, so that they begin with what pass 1 left in the 256 MB memory-side cache; ONCE (x larger
// than half of that): loads and stores that are not read again do not displace it.  32x65536x64 bf16 with residual: 227 us without
// either, 222 reversed, 186 with both; since then 122 us for this pass, 55 for pass 1, 173 in all.
template <typename T, int V, int ACT, bool ONCE> __global__ __launch_bounds__(NT) void gn_apply_kernel(FwdP p, int S2, int RS2, int join) {
    __shared__ float sm_mr[2 * JOIN_GROUPS];
    const Geo q = p.q;
    int id = gridDim.x - 1 - blockIdx.x;
    const int s = id % S2;
    id /= S2;
    const int ch = id % q.nch, b = id / q.nch;
    const int tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int c0 = ch * q.CH, c = c0 + tx * V, g0 = c0 / q.cg;
    if (join) {
        const int g1 = (min(q.C, c0 + q.CH) - 1) / q.cg, lane = tid & 63;
        for (int g = g0 + (tid >> 6); g <= g1; g += NT / 64) {
            float m, r;
            gn_join(p, b, g, lane, m, r);
            if (lane == 0) {
                sm_mr[2 * (g - g0)] = m;
                sm_mr[2 * (g - g0) + 1] = r;
                if (s == 0) {  // a group that spans chunks is written by each of them: the same value
                    p.mr[((size_t)b * q.G + g) * 2] = m;
                    p.mr[((size_t)b * q.G + g) * 2 + 1] = r;
                }
            }
        }
        __syncthreads();
    }
    if (ty >= q.R || c >= q.C) return;
    const int row0 = s * RS2, row1 = min(q.P, row0 + RS2);
    Affine<T, V, ACT> af;
    {
        float mean[V], rstd[V], mu[V], ad[V], bt[V];
        if (join) group_pairs<V>(sm_mr - 2 * g0, q.cg, c, mean, rstd);
        else group_pairs<V>(p.mr + (size_t)b * q.G * 2, q.cg, c, mean, rstd);
        affine_vec<V>(p, b, c, mu, ad, bt);
#pragma unroll
        for (int j = 0; j < V; j++) af.set(j, mean[j], mu[j] * rstd[j], ad[j]);
    }
    const int n = rows_of(row1 - row0, ty, q.R);
    const T* x = (const T*)p.x + (size_t)b * p.x_bs + (size_t)(row0 + ty) * p.x_ld + c;
    T* out = (T*)p.out + ((size_t)b * q.P + row0 + ty) * q.C + c;
    const size_t ostep = (size_t)q.R * q.C;
    if (p.res) {
        const T* res = (const T*)p.res + (size_t)b * p.r_bs + (size_t)(row0 + ty) * p.r_ld + c;
        each_row2<4, T, V, ONCE>(x, (size_t)q.R * p.x_ld, res, (size_t)q.R * p.r_ld, n, [&](const Raw<T, V>& v, const Raw<T, V>& h, int) {
            float y[V];
#pragma unroll
            for (int j = 0; j < V; j++) y[j] = af.value(j, v.get(j)) + h.get(j);
            ONCE ? vstore_once<T, V>(y, out) : vstore<T, V>(y, out);
            out += ostep;
        });
    } else {
        each_row<4, T, V, ONCE>(x, (size_t)q.R * p.x_ld, n, [&](const Raw<T, V>& v, int) {
            float y[V];
#pragma unroll
            for (int j = 0; j < V; j++) y[j] = af.value(j, v.get(j));
            ONCE ? vstore_once<T, V>(y, out) : vstore<T, V>(y, out);
            out += ostep;
        });
    }
}

// ---- one launch: a block owns an image's groups g0 .. g0 + gpc - 1 and keeps all of their pixels in registers (IPT vectors of 8
// channels per thread): x is read once, no partial sums, no second launch.  Per thread sums about its first row, as above, joined across the block.
// 32x1024x512 bf16 20.4 us = 3.3 TB/s, the reading and the writing half one after the other (every block of the launch is resident); 1x16x128 5 us, latency.
// Consecutive blocks go to the 8 XCDs in turn; the blocks of one image share 128-byte lines where a group's rows are shorter than that, so
// each XCD (and its L2) gets a contiguous run of them.  Backward 32x4096x256, 64-byte rows: 104 us in plain order, 84 so.
__device__ __forceinline__ int xcd_run(int id, int n) {
    const int per = n >> 3, extra = n & 7, x = id & 7;
    return x * per + min(x, extra) + (id >> 3);
}
constexpr int BT = 512;
struct BGeo {
    int P, C, G, cg, gpc, nch, LP, R;  // groups per block, blocks per image, vectors per row, rows at a time
};

template <typename T, int ACT, int IPT> __global__ __launch_bounds__(BT) void gn_block_kernel(FwdP p, BGeo q) {
    __shared__ float sm_mean[BT * 8], sm_m2[BT * 8];
    __shared__ float sm_mr[2 * BT];
    const int id = xcd_run(blockIdx.x, gridDim.x), b = id / q.nch, ch = id - b * q.nch, tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int g0 = ch * q.gpc, ng = min(q.gpc, q.G - g0), c0 = g0 * q.cg, CH = ng * q.cg, c = c0 + tx * 8;
    const bool on = ty < q.R && tx * 8 < CH;
    const bool whole = q.cg % 8 == 0;  // the 8 channels of a vector lie in one group: a thread has one mean, else 8
    const int pitch = whole ? q.LP : q.LP * 8;
    Raw<T, 8> f[IPT];
    const int n = on ? rows_of(q.P, ty, q.R) : 0;
    if (on) {
        const T* x = (const T*)p.x + (size_t)b * p.x_bs + (size_t)ty * p.x_ld + c;
        const size_t step = (size_t)q.R * p.x_ld;
#pragma unroll
        for (int k = 0; k < IPT; k++, x += step)
            if (k < n) f[k].load(x);
    }
    float add[8], mul[8];
    if (on) {
        float bt[8];
        affine_vec<8>(p, b, c, mul, add, bt);
        float m[8], v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) m[j] = v[j] = 0.f;
#pragma unroll
        for (int k = 1; k < IPT; k++)
            if (k < n) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float d = f[k].get(j) - f[0].get(j);
                    m[j] += d;
                    v[j] = fmaf(d, d, v[j]);
                }
            }
        if (n > 0) {
            const float inv = 1.f / (float)n;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float d = m[j] * inv;
                v[j] -= m[j] * d;
                m[j] = f[0].get(j) + d;
            }
        }
        if (whole) {
            const float all = (((m[0] + m[1]) + (m[2] + m[3])) + ((m[4] + m[5]) + (m[6] + m[7]))) * 0.125f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float d = m[j] - all;
                v[j] = fmaf((float)n * d, d, v[j]);
            }
            m[0] = all;
        }
        if (whole) {
            sm_mean[ty * pitch + tx] = m[0];
            sm_m2[ty * pitch + tx] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                sm_mean[ty * pitch + tx * 8 + j] = m[j];
                sm_m2[ty * pitch + tx * 8 + j] = v[j];
            }
        }
    }
    __syncthreads();
    const int lane = tid & 63, w = whole ? q.cg / 8 : q.cg;  // entries of a group in one row
    const double n_all = (double)q.P * (double)q.cg;
    for (int g = tid >> 6; g < ng; g += BT / 64) {
        double s = 0.0;
        for (int e = lane; e < q.R * w; e += 64) {
            const int y = e / w, n = rows_of(q.P, y, q.R);
            if (n > 0) s += (double)(n * (whole ? 8 : 1)) * (double)sm_mean[y * pitch + g * w + e - y * w];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        const double mean = s / n_all;
        double m2 = 0.0;
        for (int e = lane; e < q.R * w; e += 64) {
            const int y = e / w, n = rows_of(q.P, y, q.R);
            if (n > 0) {
                const int i = y * pitch + g * w + e - y * w;
                const double d = (double)sm_mean[i] - mean;
                m2 += (double)sm_m2[i] + (double)(n * (whole ? 8 : 1)) * d * d;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
        if (lane == 0) {
            const float mf = (float)mean, rf = (float)(1.0 / sqrt(m2 / n_all + (double)p.eps));
            sm_mr[2 * g] = mf;
            sm_mr[2 * g + 1] = rf;
            float* o = p.mr + ((size_t)b * q.G + g0 + g) * 2;
            o[0] = mf;
            o[1] = rf;
        }
    }
    __syncthreads();
    if (!on) return;
    Affine<T, 8, ACT> af;
    {
        float mean[8], rstd[8];
        group_pairs<8>(sm_mr, q.cg, tx * 8, mean, rstd);
#pragma unroll
        for (int j = 0; j < 8; j++) af.set(j, mean[j], mul[j] * rstd[j], add[j]);
    }
    const size_t rstep = (size_t)q.R * p.r_ld, ostep = (size_t)q.R * q.C;
    const T* res = p.res ? (const T*)p.res + (size_t)b * p.r_bs + (size_t)ty * p.r_ld + c : nullptr;
    T* out = (T*)p.out + ((size_t)b * q.P + ty) * q.C + c;
#pragma unroll
    for (int k = 0; k < IPT; k++) {
        if (k < n) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = af.value(j, f[k].get(j));
            if (res) {
                Raw<T, 8> h;
                h.load(res);
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] += h.get(j);
                res += rstep;
            }
            vstore<T, 8>(y, out);
            out += ostep;
        }
    }
}

// ================================================== backward ==================================================
struct BwdP {
    const void *x, *dy;
    const float *mr, *gamma, *beta, *ss;
    void* dx;
    float *dgamma, *dbeta, *dss;
    float *part;   // [B][S][C][2]: S1, S2 of a split's rows
    float *gpart;  // [B][G][nch S][2]: sums over the group's channels in the chunk of gamma' S1, gamma' S2
    float* gm;     // [B][G][2]: m1, m2, where the blocks do not join their groups themselves
    long long x_bs, x_ld, d_bs, d_ld;
    int ss_ld, ss_off, wide, B;
    Geo q;
};

// What one channel needs for du = dy act'(u), u = mul (x - mean) + add (SiLU: mul and add scaled by -log2 e)
struct ChanB {
    float mean, rstd, mul, add, tol;  // tol: below it the sign of u is not certain in fp32
};
template <int ACT, int V> __device__ __forceinline__ void chan_b(const BwdP& p, int b, int c, ChanB (&k)[V], float (&ga)[V]) {
    float mean[V], rstd[V], o[V], bt[V];
    group_pairs<V>(p.mr + (size_t)b * p.q.G * 2, p.q.cg, c, mean, rstd);
    affine_vec<V>(p, b, c, ga, o, bt);
#pragma unroll
    for (int j = 0; j < V; j++) {
        k[j].mean = mean[j];
        k[j].rstd = rstd[j];
        k[j].mul = ga[j] * rstd[j];
        k[j].add = o[j];
        k[j].tol = 1e-5f * (fabsf(bt[j]) + fabsf(o[j] - bt[j]));
        if constexpr (ACT == ACT_SILU) {
            k[j].mul *= SILU_PRE;
            k[j].add *= SILU_PRE;
        }
    }
}
// ReLU's gate within rounding distance of zero: the sign of u in fp64 from the unrounded factors.  u in fp32 is off by a few ulps of its
// terms (near zero they are as large as |beta (1 + scale)| + |shift|); a gate opened by that error would change the gradient by a whole dy.  (One value in 10^5 comes here.)
__device__ __noinline__ float relu_gate64(const float* gamma, const float* beta, const float* ss, int ss_ld, int ss_off, int b, int C, int c, float x, float mean, float rstd) {
    double a = gamma[c], o = beta[c];
    if (ss) {
        const float* row = ss + (size_t)b * ss_ld + ss_off;
        const double sc = 1.0 + (double)row[c];
        a *= sc;
        o = o * sc + (double)row[C + c];
    }
    return ((double)x - (double)mean) * (double)rstd * a + o > 0.0 ? 1.f : 0.f;
}
// xc = x - mean
template <typename T, int ACT> __device__ __forceinline__ float du_of(const BwdP& p, const ChanB& k, int b, int c, float x, float xc, float dy) {
    if constexpr (ACT == ACT_NONE) return dy;
    const float u = fmaf(xc, k.mul, k.add);
    if constexpr (ACT == ACT_RELU) {
        if (fabsf(u) <= k.tol) return dy * relu_gate64(p.gamma, p.beta, p.ss, p.ss_ld, p.ss_off, b, p.q.C, c, x, k.mean, k.rstd);
        return u > 0.f ? dy : 0.f * dy;
    } else if constexpr (ACT == ACT_SILU) {  // s (1 + v (1 - s)) for v = -ln 2 u, s = 1 / (1 + 2^u)
        const float sg = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u));
        return dy * (sg * fmaf(u, fmaf(sg, 0.69314718055994531f, -0.69314718055994531f), 1.f));
    } else {
        return dy * act_slope<T, ACT>(u);
    }
}

// ---- pass 1: per-channel sums of du and du xhat over the rows of a split.  LONG: a thread closes its sums every CHAIN rows.
template <typename T, int V, int ACT, bool LONG> __global__ __launch_bounds__(NT) void gn_bwd_sums_kernel(BwdP p) {
    using Sum = std::conditional_t<LONG, double, float>;
    __shared__ Sum sm1[NT * V], sm2[NT * V];
    const Geo q = p.q;
    int id = blockIdx.x;
    const int s = id % q.S;
    id /= q.S;
    const int ch = id % q.nch, b = id / q.nch;
    const int tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int c0 = ch * q.CH, c = c0 + tx * V;
    const int row0 = s * q.RS, row1 = min(q.P, row0 + q.RS);
    if (ty < q.R && c < q.C) {
        ChanB k[V];
        float s1[V], s2[V], ga[V];
        chan_b<ACT, V>(p, b, c, k, ga);
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
        const T* x = (const T*)p.x + (size_t)b * p.x_bs + (size_t)(row0 + ty) * p.x_ld + c;
        const T* dy = (const T*)p.dy + (size_t)b * p.d_bs + (size_t)(row0 + ty) * p.d_ld + c;
        const size_t xstep = (size_t)q.R * p.x_ld, dstep = (size_t)q.R * p.d_ld;
        const int n = rows_of(row1 - row0, ty, q.R);
        Sum *t1 = sm1 + ty * q.CH + tx * V, *t2 = sm2 + ty * q.CH + tx * V;
        for (int done = 0;;) {
            const int rows = LONG ? min(CHAIN, n - done) : n;
            each_row2<4, T, V>(x, xstep, dy, dstep, rows, [&](const Raw<T, V>& vx, const Raw<T, V>& vd, int) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xv = vx.get(j), xc = xv - k[j].mean, du = du_of<T, ACT>(p, k[j], b, c + j, xv, xc, vd.get(j));
                    s1[j] += du;
                    s2[j] = fmaf(du, xc, s2[j]);
                }
            });
#pragma unroll
            for (int j = 0; j < V; j++) {
                t1[j] = (LONG && done ? t1[j] : 0) + (Sum)s1[j];
                t2[j] = (LONG && done ? t2[j] : 0) + (Sum)(s2[j] * k[j].rstd);
                s1[j] = s2[j] = 0.f;
            }
            if (!LONG) break;
            done += rows;
            if (done >= n) break;
            x += rows * xstep;
            dy += rows * dstep;
        }
    }
    __syncthreads();
    // rows of the block, per channel; then gamma' S over the channels of each group in the chunk (gamma' S rounded to fp32 as dx_of
    // rounds gamma' du: with one value in a group both are the same number)
    for (int i = tid; i < q.CH && c0 + i < q.C; i += NT) {
        double a = 0.0, d = 0.0;
        for (int y = 0; y < q.R; y++) {
            a += (double)sm1[y * q.CH + i];
            d += (double)sm2[y * q.CH + i];
        }
        const float s1 = (float)a, s2 = (float)d;
        float* o = p.part + (((size_t)b * q.S + s) * q.C + c0 + i) * 2;
        o[0] = s1;
        o[1] = s2;
        float ga, be, sc;
        affine_of(p.gamma, p.beta, p.ss, p.ss_ld, p.ss_off, b, q.C, c0 + i, ga, be, sc);
        sm1[i] = ga * s1;  // row 0 of its own column
        sm2[i] = ga * s2;
    }
    __syncthreads();
    const int c1 = min(q.C, c0 + q.CH), g0 = c0 / q.cg, g1 = (c1 - 1) / q.cg, lane = tid & 63;
    for (int g = g0 + (tid >> 6); g <= g1; g += NT / 64) {
        const int lo = max(c0, g * q.cg) - c0, hi = min(c1, (g + 1) * q.cg) - c0;
        double a = 0.0, d = 0.0;
        for (int e = lo + lane; e < hi; e += 64) {
            a += (double)sm1[e];
            d += (double)sm2[e];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            a += __shfl_xor(a, o, 64);
            d += __shfl_xor(d, o, 64);
        }
        if (lane == 0) {
            float* o = p.gpart + (((size_t)b * q.G + g) * (q.nch * q.S) + ch * q.S + s) * 2;
            o[0] = (float)a;
            o[1] = (float)d;
        }
    }
}

// group means m1, m2 from the chunks and splits, one wave
__device__ __forceinline__ void gn_bwd_join(const BwdP& p, int b, int g, int lane, float& m1, float& m2) {
    const Geo& q = p.q;
    const int E = q.nch * q.S, ch0 = g * q.cg / q.CH, ch1 = ((g + 1) * q.cg - 1) / q.CH;  // other chunks hold nothing of the group
    const float* src = p.gpart + ((size_t)b * q.G + g) * E * 2;
    double a = 0.0, d = 0.0;
    for (int e = ch0 * q.S + lane; e < (ch1 + 1) * q.S; e += 64) {
        a += (double)src[2 * e];
        d += (double)src[2 * e + 1];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        d += __shfl_xor(d, o, 64);
    }
    const double n = (double)q.P * (double)q.cg;
    m1 = (float)(a / n);
    m2 = (float)(d / n);
}

__global__ __launch_bounds__(NT) void gn_bwd_join_kernel(BwdP p, long long n) {
    const long long i = (long long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    if (i >= n) return;
    const int b = (int)(i / p.q.G), g = (int)(i - (long long)b * p.q.G), lane = threadIdx.x & 63;
    float m1, m2;
    gn_bwd_join(p, b, g, lane, m1, m2);
    if (lane == 0) {
        p.gm[2 * i] = m1;
        p.gm[2 * i + 1] = m2;
    }
}

// S1, S2 over the splits, their gradients of scale / shift, and over the images dgamma, dbeta: a block takes 8 channels, a wave
// every fourth image, 8 lanes share the splits of a channel
__device__ void gn_bwd_params(const BwdP& p, int blk, double (*sm)[8][2]) {
    const Geo& q = p.q;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = blk * 8 + (lane & 7), si = lane >> 3;
    double ga = 0.0, gb = 0.0;
    for (int b = wave; b < p.B; b += NT / 64) {
        double a = 0.0, d = 0.0;
        if (c < q.C) {
            const float* o = p.part + ((size_t)b * q.S * q.C + c) * 2;
#pragma unroll 8
            for (int s = si; s < q.S; s += 8) {
                const f32x2 v = *reinterpret_cast<const f32x2*>(o + (size_t)s * q.C * 2);
                a += (double)v[0];
                d += (double)v[1];
            }
        }
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) {
            a += __shfl_xor(a, o, 64);
            d += __shfl_xor(d, o, 64);
        }
        const double s1 = (double)(float)a, s2 = (double)(float)d;
        double sc = 1.0;
        if (c < q.C && p.ss) {
            sc = 1.0 + (double)p.ss[(size_t)b * p.ss_ld + p.ss_off + c];
            if (si == 0 && p.dss) {
                float* o = p.dss + (size_t)b * 2 * q.C;
                o[c] = (float)((double)p.gamma[c] * s2 + (double)p.beta[c] * s1);
                o[q.C + c] = (float)s1;
            }
        }
        gb += sc * s1;
        ga += sc * s2;
    }
    if (si == 0) {
        sm[wave][lane & 7][0] = ga;
        sm[wave][lane & 7][1] = gb;
    }
    __syncthreads();
    if (tid < 8 && c < q.C) {
        for (int w = 1; w < NT / 64; w++) {
            ga += sm[w][tid][0];
            gb += sm[w][tid][1];
        }
        p.dgamma[c] = (float)ga;
        p.dbeta[c] = (float)gb;
    }
}

// rstd (g - m1 - xhat m2) with rm2 = rstd m2, xc = x - mean: the product g = gamma' du is made opaque, so that the compiler does not fuse it
// into the difference - with one value in a group, g and m1 are equal numbers and the difference has to be zero.
__device__ __forceinline__ float dx_of(float ga, float du, float rstd, float xc, float m1, float rm2) {
    float g = ga * du;
    asm volatile("" : "+v"(g));
    return rstd * ((g - m1) - xc * rm2);
}

// ---- pass 2: the first nparam blocks finish the parameters' gradients, the others write dx; as in the forward every block joins its groups itself where they
// are few (join), otherwise gn_bwd_join_kernel has (order and ONCE as in gn_apply_kernel)
template <typename T, int V, int ACT, bool ONCE> __global__ __launch_bounds__(NT) void gn_bwd_apply_kernel(BwdP p, int nparam, int S2, int RS2, int join) {
    __shared__ double sm_p[NT / 64][8][2];
    __shared__ float sm_m[2 * JOIN_GROUPS];
    if ((int)blockIdx.x < nparam) return gn_bwd_params(p, blockIdx.x, sm_p);
    const Geo q = p.q;
    int id = gridDim.x - 1 - blockIdx.x;
    const int s = id % S2;
    id /= S2;
    const int ch = id % q.nch, b = id / q.nch;
    const int tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int c0 = ch * q.CH, c = c0 + tx * V, g0 = c0 / q.cg, g1 = (min(q.C, c0 + q.CH) - 1) / q.cg, lane = tid & 63;
    if (join) {
        for (int g = g0 + (tid >> 6); g <= g1; g += NT / 64) {
            float m1, m2;
            gn_bwd_join(p, b, g, lane, m1, m2);
            if (lane == 0) {
                sm_m[2 * (g - g0)] = m1;
                sm_m[2 * (g - g0) + 1] = m2;
            }
        }
        __syncthreads();
    }
    if (ty >= q.R || c >= q.C) return;
    const int row0 = s * RS2, row1 = min(q.P, row0 + RS2);
    ChanB k[V];
    float ga[V], m1[V], m2[V];
    chan_b<ACT, V>(p, b, c, k, ga);
    if (join) group_pairs<V>(sm_m - 2 * g0, q.cg, c, m1, m2);
    else group_pairs<V>(p.gm + (size_t)b * q.G * 2, q.cg, c, m1, m2);
#pragma unroll
    for (int j = 0; j < V; j++) m2[j] *= k[j].rstd;
    const T* x = (const T*)p.x + (size_t)b * p.x_bs + (size_t)(row0 + ty) * p.x_ld + c;
    const T* dy = (const T*)p.dy + (size_t)b * p.d_bs + (size_t)(row0 + ty) * p.d_ld + c;
    T* dx = (T*)p.dx + ((size_t)b * q.P + row0 + ty) * q.C + c;
    const size_t ostep = (size_t)q.R * q.C;
    each_row2<2, T, V, ONCE>(x, (size_t)q.R * p.x_ld, dy, (size_t)q.R * p.d_ld, rows_of(row1 - row0, ty, q.R), [&](const Raw<T, V>& vx, const Raw<T, V>& vd, int) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float xv = vx.get(j), xc = xv - k[j].mean, du = du_of<T, ACT>(p, k[j], b, c + j, xv, xc, vd.get(j));
            o[j] = dx_of(ga[j], du, k[j].rstd, xc, m1[j], m2[j]);
        }
        ONCE ? vstore_once<T, V>(o, dx) : vstore<T, V>(o, dx);
        dx += ostep;
    });
}

// ---- one block per image and groups: S1, S2 of its channels, then dx.  IPT > 0: x and dy of all pixels stay in registers (IPT vectors per
// thread); IPT = 0: they are read a second time (from the cache that holds them: a block's slab is at most SLAB_MAX).
// 32x4096x256 bf16 with SiLU 75 us, 41 of them HBM's for x, dy and dx once; the slope's two quarter-rate functions per element and pass are about as much,
// and the passes follow one another.  Holding x in registers for the second pass was 3 % ahead for SiLU and spilled for ReLU and in fp32.
template <typename T, int ACT, int IPT, int NB> __global__ __launch_bounds__(NB) void gn_bwd_block_kernel(BwdP p, BGeo q) {
    __shared__ float sm1[NB * 8], sm2[NB * 8];
    __shared__ float sm_m[2 * BT];
    const int id = xcd_run(blockIdx.x, gridDim.x), b = id / q.nch, ch = id - b * q.nch, tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int g0 = ch * q.gpc, ng = min(q.gpc, q.G - g0), c0 = g0 * q.cg, CH = ng * q.cg, c = c0 + tx * 8;
    const bool on = ty < q.R && tx * 8 < CH;
    constexpr int NF = IPT > 0 ? IPT : 1;
    Raw<T, 8> fx[NF], fd[NF];
    const int n = on ? rows_of(q.P, ty, q.R) : 0;
    const T* x = (const T*)p.x + (size_t)b * p.x_bs + (size_t)ty * p.x_ld + c;
    const T* dy = (const T*)p.dy + (size_t)b * p.d_bs + (size_t)ty * p.d_ld + c;
    const size_t xstep = (size_t)q.R * p.x_ld, dstep = (size_t)q.R * p.d_ld;
    ChanB k[8];
    float ga[8];
    if (on) {
        if constexpr (IPT > 0) {
#pragma unroll
            for (int i = 0; i < IPT; i++)
                if (i < n) {
                    fx[i].load(x + i * xstep);
                    fd[i].load(dy + i * dstep);
                }
        }
        float s1[8], s2[8];
        chan_b<ACT, 8>(p, b, c, k, ga);
#pragma unroll
        for (int j = 0; j < 8; j++) s1[j] = s2[j] = 0.f;
        auto sums = [&](const Raw<T, 8>& vx, const Raw<T, 8>& vd, int) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float xv = vx.get(j), xc = xv - k[j].mean, du = du_of<T, ACT>(p, k[j], b, c + j, xv, xc, vd.get(j));
                s1[j] += du;
                s2[j] = fmaf(du, xc, s2[j]);
            }
        };
        if constexpr (IPT > 0) {
#pragma unroll
            for (int i = 0; i < IPT; i++)
                if (i < n) sums(fx[i], fd[i], i);
        } else {
            each_row2<4, T, 8>(x, xstep, dy, dstep, n, sums);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) s2[j] *= k[j].rstd;
        const int pitch = q.LP * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            sm1[ty * pitch + tx * 8 + j] = s1[j];
            sm2[ty * pitch + tx * 8 + j] = s2[j];
        }
    }
    __syncthreads();
    {   // rows: NB / CH threads per channel add every (NB / CH)-th row, then one of them joins
        const int pitch = q.LP * 8, ways = max(1, NB / CH), i = tid % CH, y0 = tid / CH;
        double a = 0.0, d = 0.0;
        if (ways > 1) {
            if (y0 < ways)
                for (int y = y0; y < q.R; y += ways) {
                    a += (double)sm1[y * pitch + i];
                    d += (double)sm2[y * pitch + i];
                }
            __syncthreads();
            if (y0 < ways && y0 < q.R) {
                sm1[y0 * CH + i] = (float)a;
                sm2[y0 * CH + i] = (float)d;
            }
            __syncthreads();
            if (tid < CH) {
                double e = 0.0, f = 0.0;
                for (int y = 0; y < min(ways, q.R); y++) {
                    e += (double)sm1[y * CH + tid];
                    f += (double)sm2[y * CH + tid];
                }
                sm1[tid] = (float)e;
                sm2[tid] = (float)f;
            }
        } else {  // a column is read and written by one thread only
            for (int c8 = tid; c8 < CH; c8 += NB) {
                a = d = 0.0;
                for (int y = 0; y < q.R; y++) {
                    a += (double)sm1[y * pitch + c8];
                    d += (double)sm2[y * pitch + c8];
                }
                sm1[c8] = (float)a;
                sm2[c8] = (float)d;
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < CH; i += NB) {
        const float t1 = sm1[i], t2 = sm2[i];
        float ga, be, sc;
        affine_of(p.gamma, p.beta, p.ss, p.ss_ld, p.ss_off, b, q.C, c0 + i, ga, be, sc);
        if (p.ss) {
            float* o = p.dss + (size_t)b * 2 * q.C + c0 + i;
            o[0] = (float)((double)p.gamma[c0 + i] * (double)t2 + (double)p.beta[c0 + i] * (double)t1);
            o[q.C] = t1;
        }
        if (p.B == 1) {
            p.dgamma[c0 + i] = t2 * sc;
            p.dbeta[c0 + i] = t1 * sc;
        } else {
            p.part[((size_t)b * q.C + c0 + i) * 2] = t1;
            p.part[((size_t)b * q.C + c0 + i) * 2 + 1] = t2;
        }
        sm1[i] = ga * t1;  // rounded as dx_of rounds gamma' du
        sm2[i] = ga * t2;
    }
    __syncthreads();
    const int lane = tid & 63;
    for (int g = tid >> 6; g < ng; g += NB / 64) {
        double a = 0.0, d = 0.0;
        for (int e = g * q.cg + lane; e < (g + 1) * q.cg; e += 64) {
            a += (double)sm1[e];
            d += (double)sm2[e];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            a += __shfl_xor(a, o, 64);
            d += __shfl_xor(d, o, 64);
        }
        const double n = (double)q.P * (double)q.cg;
        if (lane == 0) {
            sm_m[2 * g] = (float)(a / n);
            sm_m[2 * g + 1] = (float)(d / n);
        }
    }
    __syncthreads();
    if (!on) return;
    float m1[8], m2[8];
    group_pairs<8>(sm_m, q.cg, tx * 8, m1, m2);
#pragma unroll
    for (int j = 0; j < 8; j++) m2[j] *= k[j].rstd;
    T* dx = (T*)p.dx + ((size_t)b * q.P + ty) * q.C + c;
    const size_t ostep = (size_t)q.R * q.C;
    auto write = [&](const Raw<T, 8>& vx, const Raw<T, 8>& vd, int) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float xv = vx.get(j), xc = xv - k[j].mean, du = du_of<T, ACT>(p, k[j], b, c + j, xv, xc, vd.get(j));
            o[j] = dx_of(ga[j], du, k[j].rstd, xc, m1[j], m2[j]);
        }
        vstore<T, 8>(o, dx);
        dx += ostep;
    };
    if constexpr (IPT > 0) {
#pragma unroll
        for (int i = 0; i < IPT; i++)
            if (i < n) write(fx[i], fd[i], i);
    } else {
        each_row2<2, T, 8>(x, xstep, dy, dstep, n, write);
    }
}
// dgamma, dbeta from the S1, S2 that the blocks above left per image: 16 channels by 16 shares of the images, all loads of a share in flight
__global__ __launch_bounds__(256) void gn_bwd_params_kernel(BwdP p) {
    __shared__ double sm[16][16][2];
    const int cx = threadIdx.x & 15, y = threadIdx.x >> 4, C = p.q.C, c = blockIdx.x * 16 + cx;
    double ga = 0.0, gb = 0.0;
    if (c < C) {
#pragma unroll 4
        for (int b = y; b < p.B; b += 16) {
            const f32x2 v = *reinterpret_cast<const f32x2*>(p.part + ((size_t)b * C + c) * 2);
            const double sc = p.ss ? 1.0 + (double)p.ss[(size_t)b * p.ss_ld + p.ss_off + c] : 1.0;
            gb += sc * (double)v[0];
            ga += sc * (double)v[1];
        }
    }
    sm[y][cx][0] = ga;
    sm[y][cx][1] = gb;
    __syncthreads();
    if (y < 2 && c < C) {
        double t = 0.0;
#pragma unroll
        for (int k = 0; k < 16; k++) t += sm[k][cx][y];
        (y ? p.dbeta : p.dgamma)[c] = (float)t;
    }
}

// ================================================== host ==================================================
constexpr int ROWS_PER_THREAD = 8;

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int wide_params(const float* gamma, const float* beta, const float* ss, int ss_ld, int ss_off, int C) {
    return aligned16(gamma) && aligned16(beta) && (!ss || (aligned16(ss) && ss_ld % 4 == 0 && ss_off % 4 == 0 && C % 4 == 0));
}

Geo geo_any(int P, int C, int G, bool vec) { return geo_of(P, C, G, vec ? 8 : 1, ROWS_PER_THREAD); }

// Rows of a pass that needs no fixed split: about 2048 blocks in all, at least 4 rows per thread
void apply_split(const Geo& q, int B, int& S2, int& RS2) {
    long long want = 2048 / ((long long)B * q.nch);
    const long long most = (q.P + 4ll * q.R - 1) / (4ll * q.R);
    if (want > most) want = most;
    if (want < 1) want = 1;
    RS2 = (int)((q.P + want - 1) / want);
    S2 = (q.P + RS2 - 1) / RS2;
}

// The one-block form: as few whole groups per block as make 64-byte rows of whole vectors.  Returns the vectors per thread, 0 if the shape has none.
int block_geo(int P, int C, int G, int esize, BGeo& q) {
    const int cg = C / G;
    int gpc = 1;
    while (gpc < G && ((gpc * cg) % 8 != 0 || gpc * cg * esize < 64)) gpc++;
    if ((gpc * cg) % 8 != 0 || gpc * cg / 8 > BT || gpc > BT) return 0;
    q.P = P;
    q.C = C;
    q.G = G;
    q.cg = cg;
    q.gpc = gpc;
    q.nch = (G + gpc - 1) / gpc;
    q.LP = gpc * cg / 8;
    q.R = BT / q.LP;
    const long long n = ((long long)P + q.R - 1) / q.R;
    return n > (1 << 20) ? (1 << 20) : (int)n;
}
// whether every block of the last pass joins the groups of its chunk itself: few groups with few partials (a wave's round trip each)
bool joins_in_block(const Geo& q) {
    int groups = (q.CH + q.cg - 1) / q.cg + 1;  // that meet a chunk, at most
    if (groups > q.G) groups = q.G;
    return groups <= JOIN_GROUPS && (long long)groups * q.nch * q.S <= JOIN_MAX;
}
long long join_blocks(long long pairs) { return (pairs + NT / 64 - 1) / (NT / 64); }
bool read_once(long long bytes) { return bytes > (128ll << 20); }
constexpr int SLAB_BT = 512;
constexpr int SLAB_MAX = 512 << 10;  // bytes of x that one block of the backward reads twice

// whether the one-block forms take a shape of n vectors per thread
bool fwd_one_block(int n, int esize) { return n > 0 && n <= (esize == 2 ? 32 : 16); }
// The backward's takes the time of one block, whose rows every thread walks through twice, the split passes a fixed part and then that of the
// data: up to 8 vectors per thread the block is ahead for any batch.  Above, bf16: 8 x 2000x64 (16 blocks) 22.6 against 14.7 us, 8x1024x512 (64) 23.2
// against 19.0, 16x1024x512 (128) 27.0 against 27.4; slabs read twice: 32x4096x64 (64) 44 against 27, fp32 (128) 43 against 35, 32x4096x256 (256) 78
// against 86, 256x5215x16 (256) 41 against 64.
constexpr int BWD_ALWAYS = 8;
bool bwd_one_block(int n, int B, int P, const BGeo& g, int esize) {
    if (n <= BWD_ALWAYS) return n > 0;
    const long long blocks = (long long)B * g.nch;
    return n <= (esize == 2 ? 16 : 8) ? blocks >= 128 : (long long)P * g.LP * 8 * esize <= SLAB_MAX && blocks >= 192;
}

template <typename T, int ACT> int fwd_launch_vec(const FwdP& p, int B, hipStream_t st, bool& done) {
    BGeo g;
    const int n = block_geo(p.q.P, p.q.C, p.q.G, (int)sizeof(T), g);
    done = fwd_one_block(n, (int)sizeof(T));
    if (!done) return DIG_OK;
    DIG_CHECK(grid_fits((long long)B * g.nch, BT), DIG_EINVAL, "gn_act: too many blocks");
    const dim3 grid((unsigned)(B * g.nch));
    if (n <= 2) hipLaunchKernelGGL((gn_block_kernel<T, ACT, 2>), grid, dim3(BT), 0, st, p, g);
    else if (n <= 4) hipLaunchKernelGGL((gn_block_kernel<T, ACT, 4>), grid, dim3(BT), 0, st, p, g);
    else if (n <= 8) hipLaunchKernelGGL((gn_block_kernel<T, ACT, 8>), grid, dim3(BT), 0, st, p, g);
    else if (n <= 16) hipLaunchKernelGGL((gn_block_kernel<T, ACT, 16>), grid, dim3(BT), 0, st, p, g);
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((gn_block_kernel<T, ACT, 32>), grid, dim3(BT), 0, st, p, g);
    DIG_LAUNCH_CHECK("gn_act");
    return DIG_OK;
}

template <typename T, int V, int ACT> int fwd_launch(const FwdP& p, int B, hipStream_t st) {
    if constexpr (V == 8) {
        bool done;
        const int rc = fwd_launch_vec<T, ACT>(p, B, st, done);
        if (done) return rc;
    }
    const Geo& q = p.q;
    const int join = joins_in_block(q);
    DIG_CHECK(grid_fits((long long)B * q.nch * q.S, NT) && (join || grid_fits(join_blocks((long long)B * q.G), NT)), DIG_EINVAL, "gn_act: too many blocks");
    const dim3 cut((unsigned)(B * q.nch * q.S));
    if ((q.P - 1) / (q.S * q.R) >= ROWS_MAX) hipLaunchKernelGGL((gn_stats_kernel<T, V, true>), cut, dim3(NT), 0, st, p);
    else hipLaunchKernelGGL((gn_stats_kernel<T, V, false>), cut, dim3(NT), 0, st, p);
    if (!join) {
        const long long n = (long long)B * q.G;
        hipLaunchKernelGGL(gn_join_kernel, dim3((unsigned)join_blocks(n)), dim3(NT), 0, st, p, n);
    }
    int S2, RS2;
    apply_split(q, B, S2, RS2);
    const dim3 grid((unsigned)(B * q.nch * S2));
    if (V == 8 && read_once((long long)B * q.P * q.C * (long long)sizeof(T)))
        hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, true>), grid, dim3(NT), 0, st, p, S2, RS2, join);
    else hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, false>), grid, dim3(NT), 0, st, p, S2, RS2, join);
    DIG_LAUNCH_CHECK("gn_act");
    return DIG_OK;
}
template <typename T, int V> int fwd_act(const FwdP& p, int B, int act, hipStream_t st) {
    switch (act) {
        case ACT_RELU: return fwd_launch<T, V, ACT_RELU>(p, B, st);
        case ACT_GELU: return fwd_launch<T, V, ACT_GELU>(p, B, st);
        case ACT_SILU: return fwd_launch<T, V, ACT_SILU>(p, B, st);
        default: return fwd_launch<T, V, ACT_NONE>(p, B, st);
    }
}

template <typename T, int ACT> int bwd_launch_vec(BwdP p, hipStream_t st, bool& done) {
    BGeo g;
    const int n = block_geo(p.q.P, p.q.C, p.q.G, (int)sizeof(T), g);
    const int most = sizeof(T) == 2 ? 16 : 8;
    done = bwd_one_block(n, p.B, p.q.P, g, (int)sizeof(T));
    if (!done) return DIG_OK;
    DIG_CHECK(grid_fits((long long)p.B * g.nch, BT), DIG_EINVAL, "gn_act_bwd: too many blocks");
    const dim3 grid((unsigned)(p.B * g.nch));
    if (n <= 2) hipLaunchKernelGGL((gn_bwd_block_kernel<T, ACT, 2, BT>), grid, dim3(BT), 0, st, p, g);
    else if (n <= 4) hipLaunchKernelGGL((gn_bwd_block_kernel<T, ACT, 4, BT>), grid, dim3(BT), 0, st, p, g);
    else if (n <= 8) hipLaunchKernelGGL((gn_bwd_block_kernel<T, ACT, 8, BT>), grid, dim3(BT), 0, st, p, g);
    else if (n <= most) {
        if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((gn_bwd_block_kernel<T, ACT, 16, BT>), grid, dim3(BT), 0, st, p, g);
    } else {
        g.R = SLAB_BT / g.LP;
        hipLaunchKernelGGL((gn_bwd_block_kernel<T, ACT, 0, SLAB_BT>), grid, dim3(SLAB_BT), 0, st, p, g);
    }
    if (p.B > 1) {  // part is [B][C][2] here: the gradients of the parameters over the images
        hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((unsigned)((p.q.C + 15) / 16)), dim3(256), 0, st, p);
    }
    DIG_LAUNCH_CHECK("gn_act_bwd");
    return DIG_OK;
}

template <typename T, int V, int ACT> int bwd_launch(const BwdP& p, hipStream_t st) {
    if constexpr (V == 8) {
        bool done;
        const int rc = bwd_launch_vec<T, ACT>(p, st, done);
        if (done) return rc;
    }
    const Geo& q = p.q;
    int S2, RS2;
    apply_split(q, p.B, S2, RS2);
    const int nparam = (q.C + 7) / 8, join = joins_in_block(q);
    const long long pairs = (long long)p.B * q.G;
    DIG_CHECK(grid_fits((long long)p.B * q.nch * q.S, NT) && grid_fits((long long)p.B * q.nch * S2 + nparam, NT) && (join || grid_fits(join_blocks(pairs), NT)), DIG_EINVAL,
              "gn_act_bwd: too many blocks");
    const dim3 cut((unsigned)(p.B * q.nch * q.S));
    if ((q.RS - 1) / q.R >= ROWS_MAX) hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, ACT, true>), cut, dim3(NT), 0, st, p);
    else hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, ACT, false>), cut, dim3(NT), 0, st, p);
    if (!join) hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)join_blocks(pairs)), dim3(NT), 0, st, p, pairs);
    const dim3 grid((unsigned)(p.B * q.nch * S2 + nparam));
    if (V == 8 && read_once(2ll * p.B * q.P * q.C * (long long)sizeof(T)))
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, true>), grid, dim3(NT), 0, st, p, nparam, S2, RS2, join);
    else hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, false>), grid, dim3(NT), 0, st, p, nparam, S2, RS2, join);
    DIG_LAUNCH_CHECK("gn_act_bwd");
    return DIG_OK;
}
template <typename T, int V> int bwd_act(const BwdP& p, int act, hipStream_t st) {
    switch (act) {
        case ACT_RELU: return bwd_launch<T, V, ACT_RELU>(p, st);
        case ACT_GELU: return bwd_launch<T, V, ACT_GELU>(p, st);
        case ACT_SILU: return bwd_launch<T, V, ACT_SILU>(p, st);
        default: return bwd_launch<T, V, ACT_NONE>(p, st);
    }
}

bool shape_ok(int B, int P, int C, int G) { return B > 0 && P > 0 && C > 0 && G > 0 && C % G == 0 && P <= (1 << 30) && C <= (1 << 20); }

}  // namespace

extern "C" int dig_gn_act_ws(int P, int C, int groups, int bwd, int vec, int dtype) {
    if (!shape_ok(1, P, C, groups) || (vec && C % 8)) return DIG_EINVAL;
    BGeo g;
    const int esize = dtype == DIG_BF16 ? 2 : 4;
    const int per_thread = vec ? block_geo(P, C, groups, esize, g) : 0;
    if (bwd ? per_thread > 0 && per_thread <= BWD_ALWAYS : fwd_one_block(per_thread, esize)) return bwd ? C * 2 : 0;
    const Geo q = geo_any(P, C, groups, vec != 0);
    const long long n = (bwd ? 2ll * q.S * C + 2ll * groups : 0) + 2ll * groups * q.nch * q.S;
    return n < (1ll << 31) ? (int)n : DIG_EINVAL;
}

extern "C" int dig_gn_act(const dig_gn_act_args* a, void* stream) {
    DIG_CHECK(a && a->x && a->gamma && a->beta && a->out && a->mean_rstd, DIG_EINVAL, "gn_act: null pointer");
    DIG_CHECK(shape_ok(a->B, a->P, a->C, a->groups), DIG_EINVAL, "gn_act: bad shape B=%d P=%d C=%d groups=%d", a->B, a->P, a->C, a->groups);
    DIG_CHECK(a->act >= 0 && a->act <= 3, DIG_EINVAL, "gn_act: act %d", a->act);
    DIG_CHECK(a->dtype == DIG_BF16 || a->dtype == DIG_F32, DIG_EINVAL, "gn_act: dtype %d", a->dtype);
    DIG_CHECK(!a->ss || (a->ss_off >= 0 && a->ss_ld >= a->ss_off + 2 * a->C), DIG_EINVAL, "gn_act: scale/shift rows of %d values at %d do not hold 2 x %d", a->ss_ld,
              a->ss_off, a->C);
    DIG_CHECK(a->x_bs >= 0 && a->x_ld >= 0 && (!a->res || (a->res_bs >= 0 && a->res_ld >= 0)), DIG_EINVAL, "gn_act: negative pitch");
    const bool vec = a->C % 8 == 0 && a->x_bs % 8 == 0 && a->x_ld % 8 == 0 && aligned16(a->x) && aligned16(a->out) &&
                     (!a->res || (a->res_bs % 8 == 0 && a->res_ld % 8 == 0 && aligned16(a->res)));
    FwdP p{a->x, a->gamma, a->beta, a->ss, a->res, a->out, a->mean_rstd, a->ws, a->x_bs, a->x_ld, a->res_bs, a->res_ld, a->ss_ld, a->ss_off, wide_params(a->gamma, a->beta, a->ss, a->ss_ld, a->ss_off, a->C), a->eps, geo_any(a->P, a->C, a->groups, vec)};
    DIG_CHECK((long long)a->B * p.q.nch * p.q.S < (1ll << 31) && (long long)a->B * a->groups < (1ll << 31), DIG_EINVAL, "gn_act: too many blocks");
    const int need = dig_gn_act_ws(a->P, a->C, a->groups, 0, vec, a->dtype);
    DIG_CHECK(need >= 0, DIG_EINVAL, "gn_act: %d groups of %d channels need too large a workspace", a->groups, a->C);
    DIG_CHECK(need == 0 || (a->ws && aligned16(a->ws)), DIG_EINVAL, "gn_act: this shape needs a workspace, on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == DIG_BF16) return vec ? fwd_act<bf16, 8>(p, a->B, a->act, st) : fwd_act<bf16, 1>(p, a->B, a->act, st);
    return vec ? fwd_act<float, 8>(p, a->B, a->act, st) : fwd_act<float, 1>(p, a->B, a->act, st);
}

extern "C" int dig_gn_act_bwd(const dig_gn_act_bwd_args* a, void* stream) {
    DIG_CHECK(a && a->x && a->dy && a->mean_rstd && a->gamma && a->beta && a->dx && a->dgamma && a->dbeta && a->ws, DIG_EINVAL, "gn_act_bwd: null pointer");
    DIG_CHECK(shape_ok(a->B, a->P, a->C, a->groups), DIG_EINVAL, "gn_act_bwd: bad shape B=%d P=%d C=%d groups=%d", a->B, a->P, a->C, a->groups);
    DIG_CHECK(a->act >= 0 && a->act <= 3, DIG_EINVAL, "gn_act_bwd: act %d", a->act);
    DIG_CHECK(a->dtype == DIG_BF16 || a->dtype == DIG_F32, DIG_EINVAL, "gn_act_bwd: dtype %d", a->dtype);
    DIG_CHECK(!a->ss || (a->dss && a->ss_off >= 0 && a->ss_ld >= a->ss_off + 2 * a->C), DIG_EINVAL, "gn_act_bwd: scale/shift rows of %d values at %d do not hold 2 x %d",
              a->ss_ld, a->ss_off, a->C);
    const bool vec = a->C % 8 == 0 && a->x_bs % 8 == 0 && a->x_ld % 8 == 0 && a->dy_bs % 8 == 0 && a->dy_ld % 8 == 0 && aligned16(a->x) && aligned16(a->dy) &&
                     aligned16(a->dx);
    DIG_CHECK(a->x_bs >= 0 && a->x_ld >= 0 && a->dy_bs >= 0 && a->dy_ld >= 0, DIG_EINVAL, "gn_act_bwd: negative pitch");
    DIG_CHECK(dig_gn_act_ws(a->P, a->C, a->groups, 1, vec, a->dtype) >= 0, DIG_EINVAL, "gn_act_bwd: %d groups of %d channels need too large a workspace", a->groups, a->C);
    DIG_CHECK(aligned16(a->ws), DIG_EINVAL, "gn_act_bwd: ws has to lie on 16 bytes");
    const Geo q = geo_any(a->P, a->C, a->groups, vec);
    float* part = a->ws;
    float* gpart = part + (size_t)a->B * q.S * a->C * 2;
    float* gm = gpart + (size_t)a->B * a->groups * q.nch * q.S * 2;
    BwdP p{a->x, a->dy, a->mean_rstd, a->gamma, a->beta, a->ss, a->dx, a->dgamma, a->dbeta, a->dss, part, gpart, gm, a->x_bs, a->x_ld, a->dy_bs, a->dy_ld, a->ss_ld,
           a->ss_off, wide_params(a->gamma, a->beta, a->ss, a->ss_ld, a->ss_off, a->C), a->B, q};
    DIG_CHECK((long long)a->B * q.nch * q.S < (1ll << 31) && (long long)a->B * a->groups < (1ll << 31), DIG_EINVAL, "gn_act_bwd: too many blocks");
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == DIG_BF16) return vec ? bwd_act<bf16, 8>(p, a->act, st) : bwd_act<bf16, 1>(p, a->act, st);
    return vec ? bwd_act<float, 8>(p, a->act, st) : bwd_act<float, 1>(p, a->act, st);
}
