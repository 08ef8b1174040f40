// Matrix product with bias, activation and residual in its epilogue, and its backward (gfx950):
//   z = x W^T + bias,  y = act(z) [+ res];     dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz
// One MFMA tile kernel serves the three products.  It computes O[r][c] = sum_k P(r,k) Q(c,k) where either operand lies with k adjacent
// (x, W in the forward; dz in dx) or with its own index adjacent (W in dx; dz and x in dW): nothing is transposed in memory.
// The operand tiles go global -> LDS by LDS-DMA, 16 bytes a lane, in the order they lie in memory; a k-adjacent tile is read back with
// ds_read_b128, the other kind with ds_read_b64_tr_b16 (bf16: the transposing read, 4 k x 16 columns per 16 lanes) or ds_read_b32 (fp32).
// Rows of a tile all start in the same LDS bank, so 16-byte (k-adjacent) or 16-value (the other kind) slots are XORed with the row; the
// DMA writes linearly, so the swizzle is applied to the global address that a lane fetches.
// Accumulation is fp32 in the matrix units; z, act and the residual are fp32 until the one rounding of the stored value.  dz is rounded
// to the storage type once, because the matrix units take bf16 operands: half a step of bf16 per summand, of random sign, beside the
// half step of the stored dx / dW; db is summed from the unrounded dz.
#include "common.hpp"

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

__device__ __forceinline__ float act_f(int act, float u) {
    switch (act) {
        case ACT_RELU: return u < 0.f ? 0.f : u;  // keeps a NaN
        case ACT_GELU: return gelu_erf_f(u);
        case ACT_SILU: return silu_f(u);
        default: return u;
    }
}
__device__ __forceinline__ float act_d(int act, float u) {
    switch (act) {
        case ACT_RELU: return u > 0.f ? 1.f : 0.f;
        case ACT_GELU: return 0.5f * (1.f + erff(u * 0.70710678118654752f)) + u * __expf(-0.5f * u * u) * 0.39894228040143268f;
        case ACT_SILU: {
            const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-u));
            return s * (1.f + u * (1.f - s));
        }
        default: return 1.f;
    }
}

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

__device__ const f32x4 zero_piece = {0.f, 0.f, 0.f, 0.f};  // what a lane fetches for k past the end

struct LinP {
    const void *p, *q;
    long long ldp, ldq;
    int R, C, K;          // O is [R][C]
    int rpad, cpad;       // columns that exist in memory of an operand whose own index is adjacent (>= R, C)
    int kper, splits;     // k values per split (a multiple of the tile's)
    void* out;            // [R][C] row pitch ldo
    long long ldo;
    float* part;          // splits > 1: [splits][R][C] fp32
    const float* bias;
    const void* res;
    long long ldr;
    void* pre;            // z, row pitch ldo, or NULL
    int act, out_f32, vec;  // vec: 8-column vectors of out / pre / res are 16-byte aligned
};

// 8 columns of the epilogue from column c of row r: n of them exist
template <typename T> __device__ __forceinline__ void epi8(const LinP& p, float (&v)[8], int r, int c, int n) {
    const size_t o = (size_t)r * p.ldo + c;
    const T* res = p.res ? (const T*)p.res + (size_t)r * p.ldr + c : nullptr;
    T* pre = p.pre ? (T*)p.pre + o : nullptr;
    if (p.vec && n == 8) {
        if (p.bias) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += p.bias[c + j];
        }
        Frag<T> f;
        if (pre) {
#pragma unroll
            for (int j = 0; j < 8; j++) frag_set<T>(f, j, v[j]);
            frag_store<T>(f, pre);
        }
        if (p.act != ACT_NONE) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = act_f(p.act, v[j]);
        }
        if (res) {
            frag_load<T>(f, res);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += frag_get<T>(f, j);
        }
        if (p.out_f32) {
            float* d = (float*)p.out + o;
            *reinterpret_cast<f32x4*>(d) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4*>(d + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) frag_set<T>(f, j, v[j]);
            frag_store<T>(f, (T*)p.out + o);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (j < n) {
            float z = v[j] + (p.bias ? p.bias[c + j] : 0.f);
            if (pre) pre[j] = from_f32<T>(z);
            z = act_f(p.act, z);
            if (res) z += to_f32<T>(res[j]);
            if (p.out_f32) ((float*)p.out)[o + j] = z;
            else ((T*)p.out)[o + j] = from_f32<T>(z);
        }
    }
}

constexpr int KB = 128;  // bytes of k in a tile: 64 bf16 or 32 fp32 values

// One side of the tile: X rows (or columns) of the output, KB bytes of k.
template <typename T, bool TR, int X> struct Side {
    static constexpr int E = 16 / (int)sizeof(T);      // values per 16 bytes
    static constexpr int BK = KB / (int)sizeof(T);
    static constexpr int BYTES = X * KB;
    static constexpr int RB = X * (int)sizeof(T);      // row bytes of a TR tile [BK][X]
    static constexpr int GB = 16 * (int)sizeof(T);     // bytes of its 16-value slots
    static constexpr int SLOTS = X / 16;

    // swizzle of a TR tile: the rows that one read instruction takes together (bf16: 4 adjacent k in each 16-lane group, 8 apart
    // between groups; fp32: 4 apart) start in different banks
    __device__ static __forceinline__ int fk(int k) {
        if constexpr (sizeof(T) == 2) return ((k & 3) | (((k >> 3) & 1) << 2)) & (SLOTS - 1);
        else return (k >> 2) & 3 & (SLOTS - 1);
    }
    // where 16-byte piece `off` of the tile's LDS image comes from: x (row / column within the tile) and k of its first value
    __device__ static __forceinline__ void piece(int off, int& x, int& k) {
        if constexpr (TR) {
            k = off / RB;
            const int w = off - k * RB;
            x = ((w / GB) ^ fk(k)) * 16 + (w % GB) / (int)sizeof(T);
        } else {
            x = off / KB;
            k = (((off % KB) / 16) ^ (x & 7)) * E;
        }
    }
};

template <typename T> struct Ops;  // one K step of the matrix units: a fragment is what a lane holds of 16 rows
template <> struct Ops<bf16> {
    typedef bf16x8 F;
    static constexpr int KK = 32;
    __device__ static __forceinline__ void mma(f32x4& acc, const F& a, const F& b) { acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
};
template <> struct Ops<float> {
    typedef f32x4 F;
    static constexpr int KK = 16;
    __device__ static __forceinline__ void mma(f32x4& acc, const F& a, const F& b) {
#pragma unroll
        for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
    }
};

// fragment of the 16 rows from x0 (a multiple of 16), K step kk of the tile: lane l holds row l & 15, k = (l >> 4) * (KK / 4) + j
template <typename T, bool TR, int X> __device__ __forceinline__ typename Ops<T>::F frag_at(const unsigned char* t, int x0, int kk, int lane) {
    using S = Side<T, TR, X>;
    const int i = lane & 15, q = lane >> 4;
    if constexpr (!TR) {
        const int row = x0 + i;
        return *reinterpret_cast<const typename Ops<T>::F*>(t + row * KB + (((kk * 4 + q) ^ (row & 7)) * 16));
    } else if constexpr (sizeof(T) == 2) {
        s16x4 h[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int k = kk * 32 + 8 * q + 4 * u + (i >> 2);
            h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(t + k * S::RB + ((x0 / 16) ^ S::fk(k)) * S::GB + (i & 3) * 8));
        }
        const s16x8 r = {h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
        return __builtin_bit_cast(bf16x8, r);
    } else {
        f32x4 r;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int k = kk * 16 + 4 * q + j;
            r[j] = *reinterpret_cast<const float*>(t + k * S::RB + ((x0 / 16) ^ S::fk(k)) * S::GB + i * 4);
        }
        return r;
    }
}

template <int N> __device__ __forceinline__ void dma_wait_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// Tile BR x BC, WR x WC waves.  ALIGNED: both operands have 16-byte aligned rows whose k (or own index) count is a multiple of 16 bytes;
// otherwise values are fetched one by one through registers.
template <typename T, bool TP, bool TQ, int BR, int BC, int WR, int WC, bool ALIGNED>
__global__ __launch_bounds__(WR* WC * 64) void linear_kernel(LinP p, int rtiles, int ctiles) {
    using SP = Side<T, TP, BR>;
    using SQ = Side<T, TQ, BC>;
    using F = typename Ops<T>::F;
    constexpr int NW = WR * WC, BK = SP::BK, E = SP::E;
    constexpr int TRN = BR / WR / 16, TCN = BC / WC / 16;  // 16 x 16 accumulator tiles of a wave
    constexpr int WCOLS = BC / WC, OS = WCOLS + 4;
    constexpr int PCH = SP::BYTES / 1024, QCH = SQ::BYTES / 1024, STAGE = SP::BYTES + SQ::BYTES;
    constexpr int PN = PCH / NW, QN = QCH / NW;
    static_assert(PCH % NW == 0 && QCH % NW == 0, "every wave moves the same number of chunks");
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];

    // tiles to XCDs: each of the 8 gets a contiguous run of tiles (block index modulo 8 is the XCD), so that what neighbours share stays in its L2
    const int ntiles = rtiles * ctiles, id = blockIdx.x;
    int t = id % ntiles;
    const int split = id / ntiles;
    {
        const int per = ntiles / 8, extra = ntiles % 8, x = t & 7, i = t >> 3;
        t = x * per + (x < extra ? x : extra) + i;
    }
    // runs of 8 row tiles by all column tiles
    const int grp = t / (8 * ctiles), first = grp * 8, rows_in = min(8, rtiles - first), in = t - first * ctiles;
    const int r0 = (first + in % rows_in) * BR, c0 = (in / rows_in) * BC;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WC, wc = wave % WC;
    const int kbeg = split * p.kper, kend = min(p.K, kbeg + p.kper), nk = (kend - kbeg + BK - 1) / BK;

    const T* P = (const T*)p.p;
    const T* Q = (const T*)p.q;
    // this lane's pieces: element address at k tile 0, k within the tile
    const T *psrc[PN], *qsrc[QN];
    int pk[PN], qk[QN];
#pragma unroll
    for (int j = 0; j < PN; j++) {
        int x;
        SP::piece((wave + j * NW) * 1024 + lane * 16, x, pk[j]);
        if constexpr (TP) psrc[j] = P + (size_t)(kbeg + pk[j]) * p.ldp + min(r0 + x, p.rpad - (ALIGNED ? E : 1));
        else psrc[j] = P + (size_t)min(r0 + x, p.R - 1) * p.ldp + kbeg + pk[j];
    }
#pragma unroll
    for (int j = 0; j < QN; j++) {
        int x;
        SQ::piece((wave + j * NW) * 1024 + lane * 16, x, qk[j]);
        if constexpr (TQ) qsrc[j] = Q + (size_t)(kbeg + qk[j]) * p.ldq + min(c0 + x, p.cpad - (ALIGNED ? E : 1));
        else qsrc[j] = Q + (size_t)min(c0 + x, p.C - 1) * p.ldq + kbeg + qk[j];
    }
    const size_t pstep = TP ? (size_t)BK * p.ldp : (size_t)BK, qstep = TQ ? (size_t)BK * p.ldq : (size_t)BK;

    auto issue = [&](int kt, unsigned char* st) {  // k tiles are issued in order: the addresses move along
        const int left = kend - kbeg - kt * BK;    // k values left from this tile on
        const bool whole = left >= BK;
#pragma unroll
        for (int j = 0; j < PN; j++) {
            const T* s = whole || pk[j] < left ? psrc[j] : (const T*)&zero_piece;
            __builtin_amdgcn_global_load_lds((glb_void*)s, (lds_void*)(st + (wave + j * NW) * 1024), 16, 0, 0);
            psrc[j] += pstep;
        }
#pragma unroll
        for (int j = 0; j < QN; j++) {
            const T* s = whole || qk[j] < left ? qsrc[j] : (const T*)&zero_piece;
            __builtin_amdgcn_global_load_lds((glb_void*)s, (lds_void*)(st + SP::BYTES + (wave + j * NW) * 1024), 16, 0, 0);
            qsrc[j] += qstep;
        }
    };
    // unaligned operands: a piece's values one by one, zero past the end of k (and of the own index, where the next row begins)
    auto fetch = [&](int kt, unsigned char* st) {
        const int left = kend - kbeg - kt * BK;
#pragma unroll
        for (int j = 0; j < PN; j++) {
            int x, k;
            SP::piece((wave + j * NW) * 1024 + lane * 16, x, k);
            T v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool ok = TP ? k < left && r0 + x + e < p.R : k + e < left;
                v[e] = ok ? (TP ? P[(size_t)(kbeg + kt * BK + k) * p.ldp + r0 + x + e] : psrc[j][(size_t)kt * BK + e]) : from_f32<T>(0.f);
            }
#pragma unroll
            for (int e = 0; e < E; e++) reinterpret_cast<T*>(st + (wave + j * NW) * 1024 + lane * 16)[e] = v[e];
        }
#pragma unroll
        for (int j = 0; j < QN; j++) {
            int x, k;
            SQ::piece((wave + j * NW) * 1024 + lane * 16, x, k);
            T v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool ok = TQ ? k < left && c0 + x + e < p.C : k + e < left;
                v[e] = ok ? (TQ ? Q[(size_t)(kbeg + kt * BK + k) * p.ldq + c0 + x + e] : qsrc[j][(size_t)kt * BK + e]) : from_f32<T>(0.f);
            }
#pragma unroll
            for (int e = 0; e < E; e++) reinterpret_cast<T*>(st + SP::BYTES + (wave + j * NW) * 1024 + lane * 16)[e] = v[e];
        }
    };

    f32x4 acc[TRN][TCN];
#pragma unroll
    for (int i = 0; i < TRN; i++)
#pragma unroll
        for (int j = 0; j < TCN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](const unsigned char* st) {
#pragma unroll
        for (int kk = 0; kk < BK / Ops<T>::KK; kk++) {
            F fp[TRN], fq[TCN];
#pragma unroll
            for (int i = 0; i < TRN; i++) fp[i] = frag_at<T, TP, BR>(st, wr * (BR / WR) + i * 16, kk, lane);
#pragma unroll
            for (int j = 0; j < TCN; j++) fq[j] = frag_at<T, TQ, BC>(st + SP::BYTES, wc * WCOLS + j * 16, kk, lane);
#pragma unroll
            for (int i = 0; i < TRN; i++)
#pragma unroll
                for (int j = 0; j < TCN; j++) Ops<T>::mma(acc[i][j], fq[j], fp[i]);  // a lane ends with 4 adjacent columns of one row
        }
    };

    if constexpr (ALIGNED) {
        if (nk > 0) issue(0, smem);
        for (int kt = 0; kt < nk; kt++) {
            dma_wait_barrier<0>();  // tile kt is in LDS for every wave, and every wave is done with the other buffer
            if (kt + 1 < nk) issue(kt + 1, smem + ((kt + 1) & 1) * STAGE);
            compute(smem + (kt & 1) * STAGE);
        }
    } else {
        for (int kt = 0; kt < nk; kt++) {
            fetch(kt, smem);
            __syncthreads();
            compute(smem);
            __syncthreads();
        }
    }

    // ---- epilogue: 16 rows of the wave's columns at a time through its own LDS rows, then 8 adjacent columns per lane
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // the last matrix instructions have retired before their registers are read
    __syncthreads();                                     // every wave is done with the operand tiles
    float* ot = reinterpret_cast<float*>(smem) + wave * 16 * OS;
    const int i16 = lane & 15, q4 = lane >> 4;
    float* part = p.splits > 1 ? p.part + (size_t)split * p.R * p.C : nullptr;
#pragma unroll
    for (int i = 0; i < TRN; i++) {
#pragma unroll
        for (int j = 0; j < TCN; j++) *reinterpret_cast<f32x4*>(ot + i16 * OS + j * 16 + q4 * 4) = acc[i][j];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < 16 * WCOLS / 8 / 64; it++) {
            const int idx = lane + it * 64, rl = idx / (WCOLS / 8), cl = (idx % (WCOLS / 8)) * 8;
            const int r = r0 + wr * (BR / WR) + i * 16 + rl, c = c0 + wc * WCOLS + cl;
            const f32x4 a = *reinterpret_cast<const f32x4*>(ot + rl * OS + cl), b = *reinterpret_cast<const f32x4*>(ot + rl * OS + cl + 4);
            if (r < p.R && c < p.C) {
                const int n = min(8, p.C - c);
                float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
                if (part) {
                    float* d = part + (size_t)r * p.C + c;
                    if (n == 8 && p.C % 4 == 0) {
                        *reinterpret_cast<f32x4*>(d) = a;
                        *reinterpret_cast<f32x4*>(d + 4) = b;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (e < n) d[e] = v[e];
                    }
                } else {
                    epi8<T>(p, v, r, c, n);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// splits > 1: the partial products of a row's 8 columns, added in order, and the epilogue
template <typename T> __global__ __launch_bounds__(256) void linear_join_kernel(LinP p) {
    const int cv = (p.C + 7) / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)p.R * cv) return;
    const int r = (int)(i / cv), c = (int)(i - (long long)r * cv) * 8, n = min(8, p.C - c);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const float* s = p.part + (size_t)r * p.C + c;
    const size_t step = (size_t)p.R * p.C;
    if (n == 8 && p.C % 4 == 0) {
        for (int k = 0; k < p.splits; k++, s += step) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(s), b = *reinterpret_cast<const f32x4*>(s + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] += a[e];
                v[4 + e] += b[e];
            }
        }
    } else {
        for (int k = 0; k < p.splits; k++, s += step)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < n) v[e] += s[e];
    }
    epi8<T>(p, v, r, c, n);
}

// ---- dz = dy act'(z), and the column sums of the unrounded dz: a block takes 256 V columns by RPB rows
struct DzP {
    const void *dy, *pre;
    long long ldy, ldpre;
    void* dz;       // [M][ldz], columns N .. ldz - 1 zero; NULL: only the sums
    float* part;    // [row blocks][N], or NULL
    int M, N, ldz, act, rows;
};
template <typename T, int V> __global__ __launch_bounds__(256) void linear_dz_kernel(DzP p) {
    const int c = (blockIdx.x * 64 + (threadIdx.x & 63)) * V, ty = threadIdx.x >> 6;
    const int row0 = blockIdx.y * p.rows, row1 = min(p.M, row0 + p.rows), width = p.dz ? p.ldz : p.N;
    __shared__ float sm[4][64 * V + 1];
    float s[V];
#pragma unroll
    for (int j = 0; j < V; j++) s[j] = 0.f;
    if (c < width) {
        for (int r = row0 + ty; r < row1; r += 4) {
            float d[V];
            if constexpr (V == 8) {
                Frag<T> f;
                frag_load<T>(f, (const T*)p.dy + (size_t)r * p.ldy + c);
#pragma unroll
                for (int j = 0; j < 8; j++) d[j] = frag_get<T>(f, j);
                if (p.act != ACT_NONE) {
                    frag_load<T>(f, (const T*)p.pre + (size_t)r * p.ldpre + c);
#pragma unroll
                    for (int j = 0; j < 8; j++) d[j] *= act_d(p.act, frag_get<T>(f, j));
                }
                if (p.dz) {
#pragma unroll
                    for (int j = 0; j < 8; j++) frag_set<T>(f, j, d[j]);
                    frag_store<T>(f, (T*)p.dz + (size_t)r * p.ldz + c);
                }
            } else {
                d[0] = 0.f;
                if (c < p.N) {
                    d[0] = to_f32<T>(((const T*)p.dy)[(size_t)r * p.ldy + c]);
                    if (p.act != ACT_NONE) d[0] *= act_d(p.act, to_f32<T>(((const T*)p.pre)[(size_t)r * p.ldpre + c]));
                }
                if (p.dz) ((T*)p.dz)[(size_t)r * p.ldz + c] = from_f32<T>(d[0]);
            }
#pragma unroll
            for (int j = 0; j < V; j++) s[j] += d[j];
        }
    }
    if (!p.part) return;
#pragma unroll
    for (int j = 0; j < V; j++) sm[ty][(threadIdx.x & 63) * V + j] = s[j];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * V; i += 256) {
        const int col = blockIdx.x * 64 * V + i;
        if (col < p.N) p.part[(size_t)blockIdx.y * p.N + col] = (sm[0][i] + sm[1][i]) + (sm[2][i] + sm[3][i]);
    }
}
__global__ __launch_bounds__(256) void linear_db_kernel(const float* part, float* db, int chunks, int N) {
    // 16 lanes x 16 columns: 16 strides of the chunks, joined in LDS in fp64
    __shared__ double sm[16][17];
    const int cx = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + cx;
    double s = 0.0;
    if (c < N)
        for (int k = y; k < chunks; k += 16) s += (double)part[(size_t)k * N + c];
    sm[y][cx] = s;
    __syncthreads();
    if (y == 0 && c < N) {
        for (int k = 1; k < 16; k++) s += sm[k][cx];
        db[c] = (float)s;
    }
}

// ================================================== host ==================================================
inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

constexpr int TILE = 128;

// k slices of a product whose tiles do not fill the chip: about two blocks per CU, at least 4 k tiles per slice
void split_of(int R, int C, int K, int bk, int& splits, int& kper) {
    const long long tiles = (long long)((R + TILE - 1) / TILE) * ((C + TILE - 1) / TILE);
    const int nk = (K + bk - 1) / bk;
    int s = tiles >= 256 ? 1 : (int)(512 / tiles);
    if (s > nk / 4) s = nk / 4;
    if (s < 1) s = 1;
    const int per = (nk + s - 1) / s;
    splits = (nk + per - 1) / per;
    if (splits < 1) splits = 1;
    kper = per * bk;
}

template <typename T, bool TP, bool TQ, bool ALIGNED> int product_launch(LinP p, hipStream_t st) {
    constexpr int BK = KB / (int)sizeof(T);
    constexpr size_t lds = (size_t)2 * 2 * TILE * KB;  // two stages of both tiles; the epilogue's rows fit in
    static_assert(lds <= 64 * 1024, "default dynamic LDS limit");
    const int rt = (p.R + TILE - 1) / TILE, ct = (p.C + TILE - 1) / TILE;
    split_of(p.R, p.C, p.K, BK, p.splits, p.kper);
    hipLaunchKernelGGL((linear_kernel<T, TP, TQ, TILE, TILE, 2, 2, ALIGNED>), dim3((unsigned)(rt * ct * p.splits)), dim3(256), lds, st, p, rt, ct);
    if (p.splits > 1) {
        const long long n = (long long)p.R * ((p.C + 7) / 8);
        hipLaunchKernelGGL((linear_join_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
    }
    DIG_LAUNCH_CHECK("linear_act");
    return DIG_OK;
}
template <typename T, bool TP, bool TQ> int product(const LinP& p, bool aligned, hipStream_t st) {
    return aligned ? product_launch<T, TP, TQ, true>(p, st) : product_launch<T, TP, TQ, false>(p, st);
}

long long part_floats(int R, int C, int K, int dtype) {
    int s, kper;
    split_of(R, C, K, KB / (dtype == DIG_BF16 ? 2 : 4), s, kper);
    return s > 1 ? (long long)s * R * C : 0;
}

// rows of a block of the dz kernel: 128 blocks of rows, each thread at most 256 fp32 additions deep until the grid's limit
int dz_rows(int M) {
    int rows = (M + 127) / 128;
    if (rows < 32) rows = 32;
    if (rows > 1024) rows = 1024;
    if ((long long)rows * 65535 < M) rows = (int)(((long long)M + 65534) / 65535);
    return rows;
}
int dz_chunks(int M) { return (M + dz_rows(M) - 1) / dz_rows(M); }

bool shape_ok(int M, int N, int K) {
    return M > 0 && N > 0 && K > 0 && N <= (1 << 20) && K <= (1 << 20) && (long long)((M + TILE - 1) / TILE) * ((N + TILE - 1) / TILE) < (1 << 22) &&
           (long long)((M + TILE - 1) / TILE) * ((K + TILE - 1) / TILE) < (1 << 22);
}

template <typename T> int fwd(const dig_linear_act_args* a, hipStream_t st) {
    const int E = 16 / (int)sizeof(T);
    LinP p{};
    p.p = a->x;
    p.q = a->w;
    p.ldp = a->ldx;
    p.ldq = a->ldw;
    p.R = a->M;
    p.C = a->N;
    p.K = a->K;
    p.out = a->out;
    p.ldo = a->N;
    p.part = a->ws;
    p.bias = a->bias;
    p.res = a->res;
    p.ldr = a->ldr;
    p.pre = a->pre;
    p.act = a->act;
    p.vec = a->N % 8 == 0 && al16(a->out) && (!a->pre || al16(a->pre)) && (!a->res || (al16(a->res) && a->ldr % 8 == 0));
    const bool aligned = a->K % E == 0 && a->ldx % E == 0 && a->ldw % E == 0 && al16(a->x) && al16(a->w);
    return product<T, false, false>(p, aligned, st);
}

template <typename T> int bwd(const dig_linear_act_bwd_args* a, hipStream_t st) {
    const int E = 16 / (int)sizeof(T), M = a->M, N = a->N, K = a->K, ldz = (N + 7) / 8 * 8;
    const int chunks = dz_chunks(M);
    float* part = a->ws;                                    // partial products
    float* sums = a->ws + dig_linear_act_bwd_part(M, N, K, a->dtype);  // column sums of row blocks
    if (a->dz || a->db) {
        DzP d{a->dy, a->pre, a->ldy, a->ldpre, a->dz, a->db ? sums : nullptr, M, N, ldz, a->act, dz_rows(M)};
        const bool vec = N % 8 == 0 && a->ldy % 8 == 0 && al16(a->dy) && (a->act == ACT_NONE || (a->ldpre % 8 == 0 && al16(a->pre))) && (!a->dz || al16(a->dz));
        const int width = a->dz ? ldz : N;
        if (vec) hipLaunchKernelGGL((linear_dz_kernel<T, 8>), dim3((unsigned)((width + 511) / 512), (unsigned)chunks), dim3(256), 0, st, d);
        else hipLaunchKernelGGL((linear_dz_kernel<T, 1>), dim3((unsigned)((width + 63) / 64), (unsigned)chunks), dim3(256), 0, st, d);
        if (a->db) hipLaunchKernelGGL(linear_db_kernel, dim3((unsigned)((N + 15) / 16)), dim3(256), 0, st, sums, a->db, chunks, N);
        DIG_LAUNCH_CHECK("linear_act_bwd");
    }
    const void* dz = a->dz ? a->dz : a->dy;
    const long long lz = a->dz ? ldz : a->ldy;
    const bool z_ok = lz % E == 0 && al16(dz) && (a->dz || N % E == 0);
    const bool x_ok = K % E == 0 && a->ldx % E == 0 && al16(a->x), w_ok = K % E == 0 && a->ldw % E == 0 && al16(a->w);
    if (a->dx) {  // dx[m][k] = sum_n dz[m][n] W[n][k]
        LinP p{};
        p.p = dz;
        p.ldp = lz;
        p.q = a->w;
        p.ldq = a->ldw;
        p.R = M;
        p.C = p.cpad = K;
        p.K = N;
        p.out = a->dx;
        p.ldo = K;
        p.part = part;
        p.vec = K % 8 == 0 && al16(a->dx);
        const int rc = product<T, false, true>(p, z_ok && w_ok, st);
        if (rc != DIG_OK) return rc;
    }
    LinP p{};  // dW[n][k] = sum_m dz[m][n] x[m][k]
    p.p = dz;
    p.ldp = lz;
    p.q = a->x;
    p.ldq = a->ldx;
    p.R = N;
    p.rpad = a->dz ? ldz : N;
    p.C = p.cpad = K;
    p.K = M;
    p.out = a->dw;
    p.ldo = K;
    p.part = part;
    p.out_f32 = a->dw_f32;
    p.vec = K % 8 == 0 && al16(a->dw);
    return product<T, true, true>(p, z_ok && x_ok, st);
}

}  // namespace

extern "C" int dig_linear_act_ws(int M, int N, int K, int dtype) {
    if (!shape_ok(M, N, K)) return DIG_EINVAL;
    return (int)part_floats(M, N, K, dtype);
}
extern "C" int dig_linear_act_bwd_part(int M, int N, int K, int dtype) {
    if (!shape_ok(M, N, K) || !shape_ok(N, K, 1)) return DIG_EINVAL;
    const long long a = part_floats(M, K, N, dtype), b = part_floats(N, K, M, dtype);
    return (int)(((a > b ? a : b) + 3) / 4 * 4);
}
extern "C" int dig_linear_act_bwd_ws(int M, int N, int K, int dtype) {
    const int part = dig_linear_act_bwd_part(M, N, K, dtype);
    return part < 0 ? part : part + dz_chunks(M) * N;
}

extern "C" int dig_linear_act(const dig_linear_act_args* a, void* stream) {
    DIG_CHECK(a && a->x && a->w && a->out, DIG_EINVAL, "linear_act: null pointer");
    DIG_CHECK(shape_ok(a->M, a->N, a->K), DIG_EINVAL, "linear_act: bad shape M=%d N=%d K=%d", a->M, a->N, a->K);
    DIG_CHECK(a->act >= 0 && a->act <= 3, DIG_EINVAL, "linear_act: act %d", a->act);
    DIG_CHECK(a->dtype == DIG_BF16 || a->dtype == DIG_F32, DIG_EINVAL, "linear_act: dtype %d", a->dtype);
    DIG_CHECK(a->ws || dig_linear_act_ws(a->M, a->N, a->K, a->dtype) == 0, DIG_EINVAL, "linear_act: this shape needs a workspace");
    return a->dtype == DIG_BF16 ? fwd<bf16>(a, (hipStream_t)stream) : fwd<float>(a, (hipStream_t)stream);
}

extern "C" int dig_linear_act_bwd(const dig_linear_act_bwd_args* a, void* stream) {
    DIG_CHECK(a && a->x && a->w && a->dy && a->dw && a->ws, DIG_EINVAL, "linear_act_bwd: null pointer");
    DIG_CHECK(shape_ok(a->M, a->N, a->K) && shape_ok(a->N, a->K, 1), DIG_EINVAL, "linear_act_bwd: bad shape M=%d N=%d K=%d", a->M, a->N, a->K);
    DIG_CHECK(a->act >= 0 && a->act <= 3, DIG_EINVAL, "linear_act_bwd: act %d", a->act);
    DIG_CHECK(a->dtype == DIG_BF16 || a->dtype == DIG_F32, DIG_EINVAL, "linear_act_bwd: dtype %d", a->dtype);
    DIG_CHECK(a->act == ACT_NONE || (a->pre && a->dz), DIG_EINVAL, "linear_act_bwd: an activation needs pre and dz");
    return a->dtype == DIG_BF16 ? bwd<bf16>(a, (hipStream_t)stream) : bwd<float>(a, (hipStream_t)stream);
}
