// GroupNorm + scale/shift + activation + residual of a channels-last tensor (any group count), and its backward (gfx950).
//   u = gamma' (x - mean) rstd + beta',  gamma' = gamma (1 + scale_b),  beta' = beta (1 + scale_b) + shift_b,  y = act(u) [+ res]
// with mean / rstd per (image, group); the adjoint in terms of the forward's (mean, rstd):
//   du = dy act'(u),  S1[b,c] = sum_p du,  S2[b,c] = sum_p du xhat,  m1 / m2 = group means of gamma' du / gamma' du xhat,
//   dx = rstd (gamma' du - m1 - xhat m2),  dgamma = sum_b (1 + scale) S2,  dbeta = sum_b (1 + scale) S1,
//   dscale = gamma S2 + beta S1,  dshift = S1.
// Everything between the loads and the stores is fp32, sums across threads fp64; the only rounding to bf16 is the stored result.
// No atomics: partial sums lie in the workspace and are added in a fixed order, and how an image is split depends on its own
// size only, so a result does not depend on the batch it is computed in.
#include "common.hpp"

namespace {

constexpr int NT = 256;

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

template <int ACT> __device__ __forceinline__ float act_f(float u) {
    if constexpr (ACT == ACT_RELU) return u < 0.f ? 0.f : u;  // keeps a NaN
    else if constexpr (ACT == ACT_GELU) return gelu_erf_f(u);
    else if constexpr (ACT == ACT_SILU) return silu_f(u);
    else return u;
}
template <int ACT> __device__ __forceinline__ float act_d(float u) {
    if constexpr (ACT == ACT_RELU) return u > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == ACT_GELU) return 0.5f * (1.f + erff(u * 0.70710678118654752f)) + u * __expf(-0.5f * u * u) * 0.39894228040143268f;
    else if constexpr (ACT == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-u));
        return s * (1.f + u * (1.f - s));
    } else return 1.f;
}

// V consecutive channels of one row (V = 8: 16-byte aligned vectors; V = 1: any alignment)
template <typename T, int V> __device__ __forceinline__ void vload(float (&f)[V], const T* p) {
    if constexpr (V == 8) {
        Frag<T> q;
        frag_load<T>(q, p);
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = frag_get<T>(q, j);
    } else {
        f[0] = to_f32<T>(*p);
    }
}
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

// How an image is cut: chunks of channels (LP lanes x V channels), R rows at a time in a block, S splits of RS rows.
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
    if (S > 256) S = 256;
    if (S < 1) S = 1;
    q.RS = (P + S - 1) / S;
    q.S = (P + q.RS - 1) / q.RS;
    return q;
}

struct FwdP {
    const void* x;
    const float *gamma, *beta, *ss;
    const void* res;
    void* out;
    float *mr, *part;
    long long x_bs, x_ld, r_bs, r_ld;
    int ss_ld, ss_off;
    float eps;
    Geo q;
};

// ---- pass 1: (mean, M2) of every (image, group, split): per-thread sums about the thread's own first sample.  A sum of n squares
// about one of the samples is at most n + 1 times their M2, so the subtraction S2 - S1^2 / n loses at most about n ulps, whatever the mean.
template <typename T, int V> __global__ __launch_bounds__(NT) void gn_stats_kernel(FwdP p) {
    __shared__ float sm_mean[NT * V], sm_m2[NT * V];
    const Geo q = p.q;
    int id = blockIdx.x;
    const int s = id % q.S;
    id /= q.S;
    const int ch = id % q.nch, b = id / q.nch;
    const int tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int c0 = ch * q.CH, c = c0 + tx * V;
    const int row0 = s * q.RS, row1 = min(q.P, row0 + q.RS);
    const bool on = ty < q.R && c < q.C;
    const T* x = (const T*)p.x + (size_t)b * p.x_bs + c;
    float piv[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; j++) piv[j] = s1[j] = s2[j] = 0.f;
    if (on) {
        int r = row0 + ty;
        if (r < row1) vload<T, V>(piv, x + (size_t)r * p.x_ld);
        for (r += q.R; r + 3 * q.R < row1; r += 4 * q.R) {
            float f[4][V];
#pragma unroll
            for (int u = 0; u < 4; u++) vload<T, V>(f[u], x + (size_t)(r + u * q.R) * p.x_ld);
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = f[u][j] - piv[j];
                    s1[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
        }
        for (; r < row1; r += q.R) {
            float f[V];
            vload<T, V>(f, x + (size_t)r * p.x_ld);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = f[j] - piv[j];
                s1[j] += d;
                s2[j] = fmaf(d, d, s2[j]);
            }
        }
        const int len = row1 - row0, n = len > ty ? (len - ty + q.R - 1) / q.R : 0;
        const float inv = n > 0 ? 1.f / (float)n : 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float m = s1[j] * inv;
            sm_mean[ty * q.CH + tx * V + j] = piv[j] + m;
            sm_m2[ty * q.CH + tx * V + j] = s2[j] - s1[j] * m;
        }
    }
    __syncthreads();
    // groups that meet this chunk, one wave each: weighted mean, then M2 about it
    const int c1 = min(q.C, c0 + q.CH), g0 = c0 / q.cg, g1 = (c1 - 1) / q.cg, lane = tid & 63, len = row1 - row0;
    for (int g = g0 + (tid >> 6); g <= g1; g += NT / 64) {
        const int lo = max(c0, g * q.cg) - c0, hi = min(c1, (g + 1) * q.cg) - c0, w = hi - lo;
        double sn = 0.0, sm = 0.0;
        for (int e = lane; e < q.R * w; e += 64) {
            const int y = e / w, n = len > y ? (len - y + q.R - 1) / q.R : 0;
            if (n == 0) continue;
            sm += (double)n * (double)sm_mean[y * q.CH + lo + e - y * w];
            sn += (double)n;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            sm += __shfl_xor(sm, o, 64);
            sn += __shfl_xor(sn, o, 64);
        }
        const double mean = sm / sn;
        double m2 = 0.0;
        for (int e = lane; e < q.R * w; e += 64) {
            const int y = e / w, n = len > y ? (len - y + q.R - 1) / q.R : 0;
            if (n == 0) continue;
            const int i = y * q.CH + lo + e - y * w;
            const double d = (double)sm_mean[i] - mean;
            m2 += (double)sm_m2[i] + (double)n * d * d;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
        if (lane == 0) {
            float* d = p.part + (((size_t)b * q.G + g) * (q.nch * q.S) + ch * q.S + s) * 2;
            d[0] = (float)mean;
            d[1] = (float)m2;
        }
    }
}

// rows of split s times channels of group g in chunk ch
__device__ __forceinline__ double entry_count(const Geo& q, int g, int e) {
    const int ch = e / q.S, s = e - ch * q.S;
    const int rows = min(q.P, (s + 1) * q.RS) - s * q.RS;
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

// ---- pass 3: y = act(gamma' (x - mean) rstd + beta') + res
template <typename T, int V, int ACT> __global__ __launch_bounds__(NT) void gn_apply_kernel(FwdP p) {
    const Geo q = p.q;
    int id = blockIdx.x;
    const int s = id % q.S;
    id /= q.S;
    const int ch = id % q.nch, b = id / q.nch;
    const int tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int c = ch * q.CH + tx * V;
    if (ty >= q.R || c >= q.C) return;
    const int row0 = s * q.RS, row1 = min(q.P, row0 + q.RS);
    float mean[V], mul[V], add[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const float* mr = p.mr + ((size_t)b * q.G + (c + j) / q.cg) * 2;
        float sc;
        mean[j] = mr[0];
        affine_of(p.gamma, p.beta, p.ss, p.ss_ld, p.ss_off, b, q.C, c + j, mul[j], add[j], sc);
        mul[j] *= mr[1];
    }
    const T* x = (const T*)p.x + (size_t)b * p.x_bs + c;
    const T* res = p.res ? (const T*)p.res + (size_t)b * p.r_bs + c : nullptr;
    T* out = (T*)p.out + (size_t)b * q.P * q.C + c;
    for (int r = row0 + ty; r < row1; r += q.R) {
        float f[V], h[V];
        vload<T, V>(f, x + (size_t)r * p.x_ld);
        if (res) vload<T, V>(h, res + (size_t)r * p.r_ld);
#pragma unroll
        for (int j = 0; j < V; j++) {
            f[j] = act_f<ACT>(fmaf(f[j] - mean[j], mul[j], add[j]));
            if (res) f[j] += h[j];
        }
        vstore<T, V>(f, out + (size_t)r * q.C);
    }
}

// ================================================== backward ==================================================
struct BwdP {
    const void *x, *dy;
    const float *mr, *gamma, *beta, *ss;
    void* dx;
    float *dgamma, *dbeta, *dss, *part, *sums, *gm;  // part [B][S][C][2], sums [B][C][2] = (S1, S2), gm [B][G][2] = (m1, m2)
    long long x_bs, x_ld, d_bs, d_ld;
    int ss_ld, ss_off, B;
    Geo q;
};

// What one channel needs for du: u = mul (x - mean) + add.
struct ChanB {
    float mean, rstd, mul, add, tol;  // tol: below it the sign of u is not certain in fp32
};
__device__ __forceinline__ ChanB chan_b(const BwdP& p, int b, int c) {
    const float* mr = p.mr + ((size_t)b * p.q.G + c / p.q.cg) * 2;
    ChanB k;
    float sc;
    k.mean = mr[0];
    k.rstd = mr[1];
    affine_of(p.gamma, p.beta, p.ss, p.ss_ld, p.ss_off, b, p.q.C, c, k.mul, k.add, sc);
    k.mul *= k.rstd;
    k.tol = 1e-5f * (fabsf(p.beta[c] * sc) + fabsf(k.add - p.beta[c] * sc));
    return k;
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
template <int ACT> __device__ __forceinline__ float du_of(const BwdP& p, const ChanB& k, int b, int c, float x, float dy) {
    if constexpr (ACT == ACT_NONE) return dy;
    const float u = fmaf(x - k.mean, k.mul, k.add);
    if constexpr (ACT == ACT_RELU) {
        if (fabsf(u) <= k.tol) return dy * relu_gate64(p.gamma, p.beta, p.ss, p.ss_ld, p.ss_off, b, p.q.C, c, x, k.mean, k.rstd);
        return u > 0.f ? dy : 0.f * dy;
    }
    return dy * act_d<ACT>(u);
}

// ---- pass 1: per-channel sums of du and du xhat over the rows of a split
template <typename T, int V, int ACT> __global__ __launch_bounds__(NT) void gn_bwd_sums_kernel(BwdP p) {
    __shared__ float sm1[NT * V], sm2[NT * V];
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
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            k[j] = chan_b(p, b, c + j);
            s1[j] = s2[j] = 0.f;
        }
        const T* x = (const T*)p.x + (size_t)b * p.x_bs + c;
        const T* dy = (const T*)p.dy + (size_t)b * p.d_bs + c;
        for (int r = row0 + ty; r < row1; r += q.R) {
            float f[V], h[V];
            vload<T, V>(f, x + (size_t)r * p.x_ld);
            vload<T, V>(h, dy + (size_t)r * p.d_ld);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float du = du_of<ACT>(p, k[j], b, c + j, f[j], h[j]);
                s1[j] += du;
                s2[j] = fmaf(du, (f[j] - k[j].mean) * k[j].rstd, s2[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            sm1[ty * q.CH + tx * V + j] = s1[j];
            sm2[ty * q.CH + tx * V + j] = s2[j];
        }
    }
    __syncthreads();
    for (int i = tid; i < q.CH && c0 + i < q.C; i += NT) {
        double a = 0.0, d = 0.0;
        for (int y = 0; y < q.R; y++) {
            a += (double)sm1[y * q.CH + i];
            d += (double)sm2[y * q.CH + i];
        }
        float* o = p.part + (((size_t)b * q.S + s) * q.C + c0 + i) * 2;
        o[0] = (float)a;
        o[1] = (float)d;
    }
}

// ---- pass 2a: a thread per (image, channel): S1, S2 over the splits, the gradients of scale and shift
__global__ __launch_bounds__(NT) void gn_bwd_chan_kernel(BwdP p) {
    const long long i = (long long)blockIdx.x * NT + threadIdx.x;
    const Geo& q = p.q;
    if (i >= (long long)p.B * q.C) return;
    const int b = (int)(i / q.C), c = (int)(i - (long long)b * q.C);
    double a = 0.0, d = 0.0;
    for (int s = 0; s < q.S; s++) {
        const float* o = p.part + (((size_t)b * q.S + s) * q.C + c) * 2;
        a += (double)o[0];
        d += (double)o[1];
    }
    const float s1 = (float)a, s2 = (float)d;
    if (p.ss) {
        float* o = p.dss + (size_t)b * 2 * q.C;
        o[c] = fmaf(p.gamma[c], s2, p.beta[c] * s1);
        o[q.C + c] = s1;
    }
    p.sums[2 * i] = s1;
    p.sums[2 * i + 1] = s2;
}

// ---- pass 2b: waves 0 .. B G - 1: group means m1, m2; then a wave per 64 channels: dgamma, dbeta over the images
__global__ __launch_bounds__(NT) void gn_bwd_join_kernel(BwdP p) {
    const Geo& q = p.q;
    const long long w = (long long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6), ng = (long long)p.B * q.G;
    const int lane = threadIdx.x & 63;
    if (w < ng) {
        const int b = (int)(w / q.G), g = (int)(w - (long long)b * q.G);
        double a = 0.0, d = 0.0;
        for (int e = lane; e < q.cg; e += 64) {
            const int c = g * q.cg + e;
            const float* o = p.sums + ((size_t)b * q.C + c) * 2;
            // gamma' and gamma' S rounded to fp32 as dx_of rounds gamma' du: with one value in a group both are the same number
            const float ga = p.ss ? p.gamma[c] * (1.f + p.ss[(size_t)b * p.ss_ld + p.ss_off + c]) : p.gamma[c];
            float g1 = ga * o[0], g2 = ga * o[1];
            asm volatile("" : "+v"(g1), "+v"(g2));
            a += (double)g1;
            d += (double)g2;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            a += __shfl_xor(a, o, 64);
            d += __shfl_xor(d, o, 64);
        }
        const double n = (double)q.P * (double)q.cg;
        if (lane == 0) {
            p.gm[2 * w] = (float)(a / n);
            p.gm[2 * w + 1] = (float)(d / n);
        }
    } else {
        const long long c = (w - ng) * 64 + lane;
        if (c >= q.C) return;
        double a = 0.0, d = 0.0;
        for (int b = 0; b < p.B; b++) {
            const float* o = p.sums + ((size_t)b * q.C + c) * 2;
            const double sc = p.ss ? 1.0 + (double)p.ss[(size_t)b * p.ss_ld + p.ss_off + c] : 1.0;
            a += sc * (double)o[0];
            d += sc * (double)o[1];
        }
        p.dbeta[c] = (float)a;
        p.dgamma[c] = (float)d;
    }
}

// rstd (g - m1 - xhat m2): the product g = gamma' du is made opaque, so that the compiler does not fuse it into the difference - with one
// value in a group, g and m1 are equal numbers and the difference has to be zero.
__device__ __forceinline__ float dx_of(float ga, float du, float rstd, float xh, float m1, float m2) {
    float g = ga * du;
    asm volatile("" : "+v"(g));
    return rstd * ((g - m1) - xh * m2);
}

// ---- pass 3: dx
template <typename T, int V, int ACT> __global__ __launch_bounds__(NT) void gn_bwd_apply_kernel(BwdP p) {
    const Geo q = p.q;
    int id = blockIdx.x;
    const int s = id % q.S;
    id /= q.S;
    const int ch = id % q.nch, b = id / q.nch;
    const int tid = threadIdx.x, tx = tid % q.LP, ty = tid / q.LP;
    const int c = ch * q.CH + tx * V;
    if (ty >= q.R || c >= q.C) return;
    const int row0 = s * q.RS, row1 = min(q.P, row0 + q.RS);
    ChanB k[V];
    float ga[V], m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        k[j] = chan_b(p, b, c + j);
        float o, sc;
        affine_of(p.gamma, p.beta, p.ss, p.ss_ld, p.ss_off, b, q.C, c + j, ga[j], o, sc);
        const float* gm = p.gm + ((size_t)b * q.G + (c + j) / q.cg) * 2;
        m1[j] = gm[0];
        m2[j] = gm[1];
    }
    const T* x = (const T*)p.x + (size_t)b * p.x_bs + c;
    const T* dy = (const T*)p.dy + (size_t)b * p.d_bs + c;
    T* dx = (T*)p.dx + (size_t)b * q.P * q.C + c;
    for (int r = row0 + ty; r < row1; r += q.R) {
        float f[V], h[V];
        vload<T, V>(f, x + (size_t)r * p.x_ld);
        vload<T, V>(h, dy + (size_t)r * p.d_ld);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float du = du_of<ACT>(p, k[j], b, c + j, f[j], h[j]);
            f[j] = dx_of(ga[j], du, k[j].rstd, (f[j] - k[j].mean) * k[j].rstd, m1[j], m2[j]);
        }
        vstore<T, V>(f, dx + (size_t)r * q.C);
    }
}

// ================================================== host ==================================================
constexpr int ROWS_PER_THREAD = 32;

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

Geo geo_any(int P, int C, int G, bool vec) { return geo_of(P, C, G, vec ? 8 : 1, ROWS_PER_THREAD); }

template <typename T, int V> int fwd_launch(const FwdP& p, int B, int act, hipStream_t st) {
    const Geo& q = p.q;
    const dim3 grid((unsigned)(B * q.nch * q.S));
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(NT), 0, st, p);
    const long long n = (long long)B * q.G;
    hipLaunchKernelGGL(gn_join_kernel, dim3((unsigned)((n + NT / 64 - 1) / (NT / 64))), dim3(NT), 0, st, p, n);
    switch (act) {
        case ACT_RELU: hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT_RELU>), grid, dim3(NT), 0, st, p); break;
        case ACT_GELU: hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT_GELU>), grid, dim3(NT), 0, st, p); break;
        case ACT_SILU: hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT_SILU>), grid, dim3(NT), 0, st, p); break;
        default: hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT_NONE>), grid, dim3(NT), 0, st, p); break;
    }
    DIG_LAUNCH_CHECK("gn_act");
    return DIG_OK;
}

template <typename T, int V, int ACT> void bwd_launch_act(const BwdP& p, hipStream_t st) {
    const Geo& q = p.q;
    const dim3 grid((unsigned)(p.B * q.nch * q.S));
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, ACT>), grid, dim3(NT), 0, st, p);
    const long long bc = (long long)p.B * q.C, waves = (long long)p.B * q.G + (q.C + 63) / 64;
    hipLaunchKernelGGL(gn_bwd_chan_kernel, dim3((unsigned)((bc + NT - 1) / NT)), dim3(NT), 0, st, p);
    hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)((waves + NT / 64 - 1) / (NT / 64))), dim3(NT), 0, st, p);
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT>), grid, dim3(NT), 0, st, p);
}
template <typename T, int V> int bwd_launch(const BwdP& p, int act, hipStream_t st) {
    switch (act) {
        case ACT_RELU: bwd_launch_act<T, V, ACT_RELU>(p, st); break;
        case ACT_GELU: bwd_launch_act<T, V, ACT_GELU>(p, st); break;
        case ACT_SILU: bwd_launch_act<T, V, ACT_SILU>(p, st); break;
        default: bwd_launch_act<T, V, ACT_NONE>(p, st); break;
    }
    DIG_LAUNCH_CHECK("gn_act_bwd");
    return DIG_OK;
}

bool shape_ok(int B, int P, int C, int G) { return B > 0 && P > 0 && C > 0 && G > 0 && C % G == 0 && P <= (1 << 30) && C <= (1 << 20); }

}  // namespace

extern "C" int dig_gn_act_ws(int P, int C, int groups, int bwd) {
    if (!shape_ok(1, P, C, groups)) return DIG_EINVAL;
    int most = 0;
    for (int vec = 0; vec < 2; vec++) {  // whichever of the two the strides and the alignment will select
        const Geo q = geo_any(P, C, groups, vec != 0);
        const int n = bwd ? q.S * C * 2 + C * 2 + groups * 2 : groups * q.nch * q.S * 2;
        most = n > most ? n : most;
    }
    return most;
}

extern "C" int dig_gn_act(const dig_gn_act_args* a, void* stream) {
    DIG_CHECK(a && a->x && a->gamma && a->beta && a->out && a->mean_rstd && a->ws, DIG_EINVAL, "gn_act: null pointer");
    DIG_CHECK(shape_ok(a->B, a->P, a->C, a->groups), DIG_EINVAL, "gn_act: bad shape B=%d P=%d C=%d groups=%d", a->B, a->P, a->C, a->groups);
    DIG_CHECK(a->act >= 0 && a->act <= 3, DIG_EINVAL, "gn_act: act %d", a->act);
    DIG_CHECK(a->dtype == DIG_BF16 || a->dtype == DIG_F32, DIG_EINVAL, "gn_act: dtype %d", a->dtype);
    DIG_CHECK(!a->ss || (a->ss_off >= 0 && a->ss_ld >= a->ss_off + 2 * a->C), DIG_EINVAL, "gn_act: scale/shift rows of %d values at %d do not hold 2 x %d", a->ss_ld,
              a->ss_off, a->C);
    const bool vec = a->C % 8 == 0 && a->x_bs % 8 == 0 && a->x_ld % 8 == 0 && aligned16(a->x) && aligned16(a->out) &&
                     (!a->res || (a->res_bs % 8 == 0 && a->res_ld % 8 == 0 && aligned16(a->res)));
    FwdP p{a->x, a->gamma, a->beta, a->ss, a->res, a->out, a->mean_rstd, a->ws, a->x_bs, a->x_ld, a->res_bs, a->res_ld, a->ss_ld, a->ss_off, a->eps, geo_any(a->P, a->C, a->groups, vec)};
    DIG_CHECK((long long)a->B * p.q.nch * p.q.S < (1ll << 31) && (long long)a->B * a->groups < (1ll << 31), DIG_EINVAL, "gn_act: too many blocks");
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == DIG_BF16) return vec ? fwd_launch<bf16, 8>(p, a->B, a->act, st) : fwd_launch<bf16, 1>(p, a->B, a->act, st);
    return vec ? fwd_launch<float, 8>(p, a->B, a->act, st) : fwd_launch<float, 1>(p, a->B, a->act, st);
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
    const Geo q = geo_any(a->P, a->C, a->groups, vec);
    float* part = a->ws;
    float* sums = part + (size_t)a->B * q.S * a->C * 2;
    float* gm = sums + (size_t)a->B * a->C * 2;
    BwdP p{a->x, a->dy, a->mean_rstd, a->gamma, a->beta, a->ss, a->dx, a->dgamma, a->dbeta, a->dss, part, sums, gm, a->x_bs, a->x_ld, a->dy_bs, a->dy_ld, a->ss_ld,
           a->ss_off, a->B, q};
    DIG_CHECK((long long)a->B * q.nch * q.S < (1ll << 31) && (long long)a->B * a->groups < (1ll << 31), DIG_EINVAL, "gn_act_bwd: too many blocks");
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == DIG_BF16) return vec ? bwd_launch<bf16, 8>(p, a->act, st) : bwd_launch<bf16, 1>(p, a->act, st);
    return vec ? bwd_launch<float, 8>(p, a->act, st) : bwd_launch<float, 1>(p, a->act, st);
}
