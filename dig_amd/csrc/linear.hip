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
#include <type_traits>

#include "act.hpp"

namespace {

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

// 8 columns of the epilogue from column c of row r: n of them exist.  FULL: bias, pre, act and res; otherwise only the store.  rv: the
// residual's vector, if p.vec
template <typename T, int ACT, bool FULL> __device__ __forceinline__ void epi8(const LinP& p, float (&v)[8], int r, int c, int n, const Frag<T>& rv) {
    const size_t o = (size_t)r * p.ldo + c;
    if (p.vec) {  // n is 8
        Frag<T> f;
        if constexpr (FULL) {
            if (p.bias) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] += p.bias[c + j];
            }
            if (p.pre) {
#pragma unroll
                for (int j = 0; j < 8; j++) frag_set<T>(f, j, v[j]);
                frag_store<T>(f, (T*)p.pre + o);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = act_val<T, ACT>(v[j]);
            if (p.res) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] += frag_get<T>(rv, j);
            }
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
            float z = v[j];
            if constexpr (FULL) {
                if (p.bias) z += p.bias[c + j];
                if (p.pre) ((T*)p.pre)[o + j] = from_f32<T>(z);
                z = act_val<T, ACT>(z);
                if (p.res) z += to_f32<T>(((const T*)p.res)[(size_t)r * p.ldr + c + j]);
            }
            if (p.out_f32) ((float*)p.out)[o + j] = z;
            else ((T*)p.out)[o + j] = from_f32<T>(z);
        }
    }
}

typedef std::integral_constant<bool, true> yes;
typedef std::integral_constant<bool, false> no;

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
// otherwise values are fetched one by one through registers.  FULL: the forward's epilogue.
//
// A wave holds the fragments of two K steps: those of the next step are read between the matrix instructions of this one (the order is
// pinned with sched_barrier: left alone, hipcc sinks the reads to their first use).  One barrier per tile of 128 bytes of k, before its
// last K step: by then the wave holds the rest of the tile in registers, and the next tile is in LDS.
// Both operands k-adjacent: NS tiles in LDS, filled by LDS-DMA; the place of a tile is filled again during its last K step.
// Otherwise (TQ): two tiles in LDS, filled through registers, which fetch a tile ahead - hipcc waits for every DMA in flight before a transposing
// read, so the two do not go together.
template <typename T, bool TP, bool TQ, int BR, int BC, int WR, int WC, int NS, bool ALIGNED, bool FULL>
__global__ __launch_bounds__(WR* WC * 64, BR * BC <= 128 * 128 || WR * WC == 8 ? 2 : 1) void linear_kernel(LinP p, int rtiles, int ctiles) {
    using SP = Side<T, TP, BR>;
    using SQ = Side<T, TQ, BC>;
    using F = typename Ops<T>::F;
    constexpr int NW = WR * WC, BK = SP::BK, E = SP::E, KKN = BK / Ops<T>::KK;
    constexpr int TRN = BR / WR / 16, TCN = BC / WC / 16;  // 16 x 16 accumulator tiles of a wave
    constexpr int WCOLS = BC / WC, OS = WCOLS + 4;
    constexpr int PCH = SP::BYTES / 1024, QCH = SQ::BYTES / 1024, STAGE = SP::BYTES + SQ::BYTES;
    constexpr int PN = PCH / NW, QN = QCH / NW;
    static_assert(PCH % NW == 0 && QCH % NW == 0, "every wave moves the same number of chunks");
    static_assert(KKN == 2, "two sets of fragments");
    constexpr bool STAGED = TQ;
    static_assert(!STAGED || NS == 2, "two tiles");
    static_assert(TRN >= 2, "rows to spread the reads over");
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

    const T* P = (const T*)p.p + (TP ? (size_t)kbeg * p.ldp + r0 : (size_t)r0 * p.ldp + kbeg);
    const T* Q = (const T*)p.q + (TQ ? (size_t)kbeg * p.ldq + c0 : (size_t)c0 * p.ldq + kbeg);

    f32x4 acc[TRN][TCN];
#pragma unroll
    for (int i = 0; i < TRN; i++)
#pragma unroll
        for (int j = 0; j < TCN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto pfrag = [&](const unsigned char* st, int i, int kk) { return frag_at<T, TP, BR>(st, wr * (BR / WR) + i * 16, kk, lane); };
    auto qfrag = [&](const unsigned char* st, int j, int kk) { return frag_at<T, TQ, BC>(st + SP::BYTES, wc * WCOLS + j * 16, kk, lane); };

    if constexpr (ALIGNED) {
        // this lane's pieces: byte offset from the tile's corner at its first k (the host checks that it fits in 31 bits), k within the tile
        unsigned poff[PN], qoff[QN];
        int pk[PN], qk[QN];
#pragma unroll
        for (int j = 0; j < PN; j++) {
            int x;
            SP::piece((wave + j * NW) * 1024 + lane * 16, x, pk[j]);
            poff[j] = (TP ? (unsigned)pk[j] * (unsigned)p.ldp + min(x, p.rpad - E - r0) : (unsigned)min(x, p.R - 1 - r0) * (unsigned)p.ldp + pk[j]) * (unsigned)sizeof(T);
        }
#pragma unroll
        for (int j = 0; j < QN; j++) {
            int x;
            SQ::piece((wave + j * NW) * 1024 + lane * 16, x, qk[j]);
            qoff[j] = (TQ ? (unsigned)qk[j] * (unsigned)p.ldq + min(x, p.cpad - E - c0) : (unsigned)min(x, p.C - 1 - c0) * (unsigned)p.ldq + qk[j]) * (unsigned)sizeof(T);
        }
        const size_t pstep = (TP ? (size_t)BK * p.ldp : (size_t)BK) * sizeof(T), qstep = (TQ ? (size_t)BK * p.ldq : (size_t)BK) * sizeof(T);
        const char *pb = (const char*)P, *qb = (const char*)Q;  // k tiles are issued in order: the corners move along
        int left = kend - kbeg;                                 // k values from the next tile to issue on
        // where the j-th of the wave's PN + QN chunks comes from; past the end of k, also behind the last tile, from zeros
        auto source = [&](int j) {
            const bool is_p = j < PN;
            const int i = is_p ? j : j - PN;
            const char* src = is_p ? pb + poff[is_p ? i : 0] : qb + qoff[is_p ? 0 : i];
            return (is_p ? pk[is_p ? i : 0] : qk[is_p ? 0 : i]) < left ? src : (const char*)&zero_piece;
        };
        auto place1 = [&](int j, unsigned char* st) { return st + (j < PN ? 0 : SP::BYTES) + (wave + (j < PN ? j : j - PN) * NW) * 1024; };
        auto issue1 = [&](int j, unsigned char* st) { __builtin_amdgcn_global_load_lds((glb_void*)source(j), (lds_void*)place1(j, st), 16, 0, 0); };
        auto advance = [&]() {
            pb += pstep;
            qb += qstep;
            left -= BK;
        };
        f32x4 rg[STAGED ? PN + QN : 1];
        auto fetch = [&]() {  // a tile into registers
#pragma unroll
            for (int j = 0; j < PN + QN; j++) rg[STAGED ? j : 0] = *reinterpret_cast<const f32x4*>(source(j));
            advance();
        };
        auto put1 = [&](int j, unsigned char* st) { *reinterpret_cast<f32x4*>(place1(j, st) + lane * 16) = rg[STAGED ? j : 0]; };
        F fp[2][TRN], fq[2][TCN];
        if constexpr (STAGED) {
            fetch();
#pragma unroll
            for (int j = 0; j < PN + QN; j++) put1(j, smem);
            fetch();
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < NS; i++) {
#pragma unroll
                for (int j = 0; j < PN + QN; j++) issue1(j, smem + i * STAGE);
                advance();
            }
            dma_wait_barrier<(NS - 1) * (PN + QN)>();
        }
#pragma unroll
        for (int j = 0; j < TCN; j++) fq[0][j] = qfrag(smem, j, 0);
#pragma unroll
        for (int i = 0; i < TRN; i++) fp[0][i] = pfrag(smem, i, 0);
        unsigned char *cur = smem, *nxt = smem + STAGE;
        // one copy of the matrix instructions and no branch in it: behind the last tile, tiles of zeros are fetched and not used
        for (int kt = 0; kt < nk; kt++) {
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                const unsigned char* from = kk ? nxt : cur;
                if (kk) {
                    if constexpr (STAGED) {
                        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    } else {
                        dma_wait_barrier<(NS - 2) * (PN + QN)>();  // the next tile has landed; those behind it may be on their way
                    }
                }
#pragma unroll
                for (int i = 0; i < TRN; i++) {
#pragma unroll
                    for (int j = 0; j < TCN; j++) Ops<T>::mma(acc[i][j], fq[kk][j], fp[kk][i]);  // a lane ends with 4 adjacent columns of one row
                    __builtin_amdgcn_sched_barrier(0);
                    if (i < TRN - 1) {  // the next step's fragments, spread over the rows of this one but the last, which covers their latency
#pragma unroll
                        for (int e = i * (TRN + TCN) / (TRN - 1); e < (i + 1) * (TRN + TCN) / (TRN - 1); e++) {
                            if (e < TCN) fq[kk ^ 1][e < TCN ? e : 0] = qfrag(from, e, kk ^ 1);
                            else fp[kk ^ 1][e < TCN ? 0 : e - TCN] = pfrag(from, e - TCN, kk ^ 1);
                        }
                    }
                    if constexpr (STAGED) {
                        if (kk == 0) {
#pragma unroll
                            for (int e = i * (PN + QN) / TRN; e < (i + 1) * (PN + QN) / TRN; e++) put1(e, nxt);
                            if (i == TRN - 1) fetch();
                        }
                    } else if (kk == 1) {  // a few at a time: a burst of them stalls the wave
#pragma unroll
                        for (int e = i * (PN + QN) / TRN; e < (i + 1) * (PN + QN) / TRN; e++) issue1(e, cur);
                        if (i == TRN - 1) advance();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            cur = nxt;
            nxt = cur == smem + (NS - 1) * STAGE ? smem : cur + STAGE;
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the last of them have landed before LDS is used again
    } else {
        // a piece's values one by one, zero past the end of k (and of the own index, where the next row begins)
        auto fetch = [&](const T* X, long long ld, int off, int x, int k, bool tr, int lim, int left, unsigned char* st) {
            T v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool ok = tr ? k < left && x + e < lim : k + e < left && x < lim;
                v[e] = ok ? X[tr ? (size_t)k * ld + x + e : (size_t)x * ld + k + e] : from_f32<T>(0.f);
            }
#pragma unroll
            for (int e = 0; e < E; e++) reinterpret_cast<T*>(st + off)[e] = v[e];
        };
        for (int kt = 0; kt < nk; kt++) {
            const int left = kend - kbeg - kt * BK;
#pragma unroll
            for (int j = 0; j < PN; j++) {
                const int off = (wave + j * NW) * 1024 + lane * 16;
                int x, k;
                SP::piece(off, x, k);
                fetch(P + (TP ? (size_t)kt * BK * p.ldp : (size_t)kt * BK), p.ldp, off, x, k, TP, p.R - r0, left, smem);
            }
#pragma unroll
            for (int j = 0; j < QN; j++) {
                const int off = (wave + j * NW) * 1024 + lane * 16;
                int x, k;
                SQ::piece(off, x, k);
                fetch(Q + (TQ ? (size_t)kt * BK * p.ldq : (size_t)kt * BK), p.ldq, off, x, k, TQ, p.C - c0, left, smem + SP::BYTES);
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                F fp[TRN], fq[TCN];
#pragma unroll
                for (int i = 0; i < TRN; i++) fp[i] = pfrag(smem, i, kk);
#pragma unroll
                for (int j = 0; j < TCN; j++) fq[j] = qfrag(smem, j, kk);
#pragma unroll
                for (int i = 0; i < TRN; i++)
#pragma unroll
                    for (int j = 0; j < TCN; j++) Ops<T>::mma(acc[i][j], fq[j], fp[i]);
            }
            __syncthreads();
        }
    }

    // ---- epilogue: 16 rows of the wave's columns at a time through its own LDS rows, then 8 adjacent columns per lane.  The residual of
    // the next 16 rows is fetched while these are worked on.
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // the last matrix instructions have retired before their registers are read
    __syncthreads();                                     // every wave is done with the operand tiles
    float* ot = reinterpret_cast<float*>(smem) + wave * 16 * OS;
    const int i16 = lane & 15, q4 = lane >> 4;
    constexpr int ITEMS = 16 * WCOLS / 8 / 64;
    static_assert(ITEMS >= 1, "a wave has at least 32 columns");
    float* part = p.splits > 1 ? p.part + (size_t)split * p.R * p.C : nullptr;
    const bool use_res = FULL && p.res && p.vec && !part;
    auto place = [&](int i, int it, int& r, int& c) {
        const int idx = lane + it * 64;
        r = r0 + wr * (BR / WR) + i * 16 + idx / (WCOLS / 8);
        c = c0 + wc * WCOLS + (idx % (WCOLS / 8)) * 8;
    };
    Frag<T> rn[ITEMS];
    auto fetch_res = [&](int i) {
#pragma unroll
        for (int it = 0; it < ITEMS; it++) {
            int r, c;
            place(i, it, r, c);
            if (r < p.R && c < p.C) frag_load<T>(rn[it], (const T*)p.res + (size_t)r * p.ldr + c);
        }
    };
    auto finish = [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (use_res) fetch_res(0);
#pragma unroll
        for (int i = 0; i < TRN; i++) {
#pragma unroll
            for (int j = 0; j < TCN; j++) *reinterpret_cast<f32x4*>(ot + i16 * OS + j * 16 + q4 * 4) = acc[i][j];
            __builtin_amdgcn_wave_barrier();
            Frag<T> rv[ITEMS];
#pragma unroll
            for (int it = 0; it < ITEMS; it++) rv[it] = rn[it];
            if (use_res && i + 1 < TRN) fetch_res(i + 1);
#pragma unroll
            for (int it = 0; it < ITEMS; it++) {
                const int idx = lane + it * 64, rl = idx / (WCOLS / 8), cl = (idx % (WCOLS / 8)) * 8;
                int r, c;
                place(i, it, r, c);
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
                        epi8<T, ACT, FULL>(p, v, r, c, n, rv[it]);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    };
    if constexpr (FULL) {
        if (p.act == ACT_RELU) finish(std::integral_constant<int, ACT_RELU>());
        else if (p.act == ACT_GELU) finish(std::integral_constant<int, ACT_GELU>());
        else if (p.act == ACT_SILU) finish(std::integral_constant<int, ACT_SILU>());
        else finish(std::integral_constant<int, ACT_NONE>());
    } else {
        finish(std::integral_constant<int, ACT_NONE>());
    }
}

// splits > 1: the partial products of a row's 8 columns, added in order, and the epilogue
template <typename T, int ACT, bool FULL> __global__ __launch_bounds__(256) void linear_join_kernel(LinP p) {
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
    Frag<T> rv;
    if (FULL && p.res && p.vec) frag_load<T>(rv, (const T*)p.res + (size_t)r * p.ldr + c);
    epi8<T, ACT, FULL>(p, v, r, c, n, rv);
}

// ---- dz = dy act'(z), and the column sums of the unrounded dz: a block takes 256 V columns by RPB rows
struct DzP {
    const void *dy, *pre;
    long long ldy, ldpre;
    void* dz;       // [M][ldz], columns N .. ldz - 1 zero; NULL: only the sums
    float* part;    // [row blocks][N], or NULL
    int M, N, ldz, rows;
};
template <typename T, int V, int ACT> __global__ __launch_bounds__(256) void linear_dz_kernel(DzP p) {
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
                if constexpr (ACT != ACT_NONE) {
                    frag_load<T>(f, (const T*)p.pre + (size_t)r * p.ldpre + c);
#pragma unroll
                    for (int j = 0; j < 8; j++) d[j] *= act_slope<T, ACT>(frag_get<T>(f, j));
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
                    if constexpr (ACT != ACT_NONE) d[0] *= act_slope<T, ACT>(to_f32<T>(((const T*)p.pre)[(size_t)r * p.ldpre + c]));
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
#ifndef BIG_TILE
#define BIG_TILE 0
#define BT_R 256
#define BT_C 256
#define BT_WR 2
#define BT_WC 2
#define BT_NS 2
#endif

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

template <typename T, bool FULL> void join_launch(const LinP& p, hipStream_t st) {
    const long long n = (long long)p.R * ((p.C + 7) / 8);
    const dim3 grid((unsigned)((n + 255) / 256));
    if constexpr (FULL) {
        switch (p.act) {
            case ACT_RELU: hipLaunchKernelGGL((linear_join_kernel<T, ACT_RELU, true>), grid, dim3(256), 0, st, p); return;
            case ACT_GELU: hipLaunchKernelGGL((linear_join_kernel<T, ACT_GELU, true>), grid, dim3(256), 0, st, p); return;
            case ACT_SILU: hipLaunchKernelGGL((linear_join_kernel<T, ACT_SILU, true>), grid, dim3(256), 0, st, p); return;
            default: break;
        }
    }
    hipLaunchKernelGGL((linear_join_kernel<T, ACT_NONE, FULL>), grid, dim3(256), 0, st, p);
}

template <typename T, bool TP, bool TQ, int BR, int BC, int WR, int WC, int NS, bool ALIGNED> int tile_launch(const LinP& p, hipStream_t st) {
    constexpr bool FULL = !TQ;  // the forward
    constexpr size_t stages = (size_t)(ALIGNED ? NS : 1) * (BR + BC) * KB, rows = (size_t)WR * WC * 16 * (BC / WC + 4) * 4, lds = stages > rows ? stages : rows;
    auto kern = linear_kernel<T, TP, TQ, BR, BC, WR, WC, NS, ALIGNED, FULL>;
    if constexpr (lds > 64 * 1024) {
        static std::atomic<bool> attr_set[64];
        int dev = 0;
        (void)hipGetDevice(&dev);
        dev &= 63;
        if (!attr_set[dev].load(std::memory_order_acquire)) {
            const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            DIG_CHECK(e == hipSuccess, DIG_ELAUNCH, "linear_act: cannot raise dynamic LDS to %zu: %s", lds, hipGetErrorString(e));
            attr_set[dev].store(true, std::memory_order_release);
        }
    }
    const int rt = (p.R + BR - 1) / BR, ct = (p.C + BC - 1) / BC;
    hipLaunchKernelGGL(kern, dim3((unsigned)(rt * ct * p.splits)), dim3(WR * WC * 64), lds, st, p, rt, ct);
    if (p.splits > 1) join_launch<T, FULL>(p, st);
    DIG_LAUNCH_CHECK("linear_act");
    return DIG_OK;
}

template <typename T, bool TP, bool TQ> int product(LinP p, bool aligned, hipStream_t st) {
    constexpr int BK = KB / (int)sizeof(T);
    split_of(p.R, p.C, p.K, BK, p.splits, p.kper);
#ifdef NOSPLIT
    p.splits = 1; p.kper = (p.K + BK - 1) / BK * BK;
#endif
    // byte offsets inside a tile are 31 bits: 256 rows of k-adjacent operands, BK rows of the others
    const long long po = (long long)(TP ? BK : 256) * p.ldp, qo = (long long)(TQ ? BK : 256) * p.ldq;
    if (po * (long long)sizeof(T) >= (1ll << 31) || qo * (long long)sizeof(T) >= (1ll << 31)) aligned = false;
    if (!aligned) return tile_launch<T, TP, TQ, 128, 128, 2, 2, 2, false>(p, st);
    if (BIG_TILE) return tile_launch<T, TP, TQ, BT_R, BT_C, BT_WR, BT_WC, (TQ ? 2 : BT_NS), true>(p, st);
    return tile_launch<T, TP, TQ, 128, 128, 2, 2, 2, true>(p, st);
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

template <typename T, int ACT> void dz_launch(const DzP& d, bool vec, dim3 grid, hipStream_t st) {
    if (vec) hipLaunchKernelGGL((linear_dz_kernel<T, 8, ACT>), grid, dim3(256), 0, st, d);
    else hipLaunchKernelGGL((linear_dz_kernel<T, 1, ACT>), grid, dim3(256), 0, st, d);
}

template <typename T> int bwd(const dig_linear_act_bwd_args* a, hipStream_t st) {
    const int E = 16 / (int)sizeof(T), M = a->M, N = a->N, K = a->K, ldz = (N + 7) / 8 * 8;
    const int chunks = dz_chunks(M);
    float* part = a->ws;                                    // partial products
    float* sums = a->ws + dig_linear_act_bwd_part(M, N, K, a->dtype);  // column sums of row blocks
    if (a->dz || a->db) {
        DzP d{a->dy, a->pre, a->ldy, a->ldpre, a->dz, a->db ? sums : nullptr, M, N, ldz, dz_rows(M)};
        const bool vec = N % 8 == 0 && a->ldy % 8 == 0 && al16(a->dy) && (a->act == ACT_NONE || (a->ldpre % 8 == 0 && al16(a->pre))) && (!a->dz || al16(a->dz));
        const int width = a->dz ? ldz : N;
        const dim3 grid((unsigned)(vec ? (width + 511) / 512 : (width + 63) / 64), (unsigned)chunks);
        switch (a->act) {
            case ACT_RELU: dz_launch<T, ACT_RELU>(d, vec, grid, st); break;
            case ACT_GELU: dz_launch<T, ACT_GELU>(d, vec, grid, st); break;
            case ACT_SILU: dz_launch<T, ACT_SILU>(d, vec, grid, st); break;
            default: dz_launch<T, ACT_NONE>(d, vec, grid, st); break;
        }
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
