// Matrix product with bias, activation and residual in its epilogue, and its backward (gfx950):
//   z = x W^T + bias,  y = act(z) [+ res];     dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz
// One MFMA tile kernel serves the three products.  It computes O[r][c] = sum_k P(r,k) Q(c,k) where either operand lies with k adjacent
// (x, W in the forward; dz in dx) or with its own index adjacent (W in dx; dz and x in dW): nothing is transposed in memory.
// The operand tiles go to LDS 16 bytes a lane in the order they lie in memory (by LDS-DMA in the forward, through registers in the backward); a
// k-adjacent tile is read back with ds_read_b128, the other kind with ds_read_b64_tr_b16 (bf16: the transposing read, 4 k x 16 columns per 16
// lanes) or ds_read_b32 (fp32).  Rows of a tile all start in the same LDS bank, so 16-byte (k-adjacent) or 16-value (the other kind) slots are
// XORed with the row; LDS is written linearly, so the swizzle is applied to the global address that a lane fetches.
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

template <bool FULL> __device__ __forceinline__ void load_bias(const LinP& p, int c, float (&bias)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) bias[j] = FULL && p.bias && c + j < p.C ? p.bias[c + j] : 0.f;
}

// 8 columns of the epilogue from column c of row r (p.vec).  FULL: bias, pre, act and res; otherwise only the store.  rv: the residual's vector
template <typename T, int ACT, bool FULL> __device__ __forceinline__ void epi8(const LinP& p, float (&v)[8], int r, int c, const Frag<T>& rv, const float (&bias)[8]) {
    const size_t o = (size_t)r * p.ldo + c;
    Frag<T> f;
    if constexpr (FULL) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] += bias[j];
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
}
// one value, where rows do not start on 16 bytes
template <typename T, int ACT, bool FULL> __device__ __forceinline__ void epi1(const LinP& p, float z, int r, int c) {
    const size_t o = (size_t)r * p.ldo + c;
    if constexpr (FULL) {
        if (p.bias) z += p.bias[c];
        if (p.pre) ((T*)p.pre)[o] = from_f32<T>(z);
        z = act_val<T, ACT>(z);
        if (p.res) z += to_f32<T>(((const T*)p.res)[(size_t)r * p.ldr + c]);
    }
    if (p.out_f32) ((float*)p.out)[o] = z;
    else ((T*)p.out)[o] = from_f32<T>(z);
}

// f(0), ..., f(N - 1) with constant indices: hipcc gives up on unrolling a large body, and an array of accumulators indexed by a variable goes to memory
template <int N, typename F> __device__ __forceinline__ void static_for(F&& f) {
    if constexpr (N > 0) {
        static_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>());
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

// Bound by the matrix units where k is long: 8192x4096x4096 bf16 with SiLU and residual 239 us = 1.15 PFLOP/s, 223 on inputs that stay in the caches (a library
// product of that size alone takes 203 us); fp32 127 TFLOP/s at 2048x2048x2048, 113 at 6272x4096x1024 and 95 at 6912x384x1536, of the 154 that a large library
// product reaches.  The fp32 backward of 5864x1536x384 makes 100 TFLOP/s, its matrix units busy in 80 % of the CUs' busy cycles.  With few k tiles the first
// tile's latency and the epilogue's stores are most of it: 6912x1536x384 with GELU and pre 22 us (24 traced), of which the bytes are 10.
// Tile BR x BC, WR x WC waves.  Both operands have 16-byte aligned rows whose k (or own index) count fills them (the host packs others first).
// FULL: the forward's epilogue.
//
// A wave holds the fragments of two K steps: those of the next step are read between the matrix instructions of this one (the order is
// pinned with sched_barrier: left alone, hipcc sinks the reads to their first use).  One barrier per tile of 128 bytes of k, before its
// last K step: by then the wave holds the rest of the tile in registers, and the next tile is in LDS.
// Both operands k-adjacent: NS tiles in LDS, filled by LDS-DMA; the place of a tile is filled again during its last K step.
// Otherwise (TQ): two tiles in LDS, filled through registers, which fetch a tile ahead: with the builtin for LDS-DMA hipcc waits for every DMA in flight
// before a transposing read (a DMA issued from inline asm, which it does not track, has not been tried here).
template <typename T, bool TP, bool TQ, int BR, int BC, int WR, int WC, int NS, bool FULL>
__device__ __forceinline__ void linear_tile(const LinP& p, int rtiles, int ctiles, int id, unsigned char* smem) {
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
    // tiles to XCDs: each of the 8 gets a contiguous run of tiles (block index modulo 8 is the XCD), so that what neighbours share stays in its L2
    const int ntiles = rtiles * ctiles;
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

    {
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
        // Order of the k tiles: a partial one at the end of k goes first, with its pieces past the end replaced by zeros; the whole ones follow from the
        // corner on.  So the loop fetches without a mask, from a scalar base that moves along and a fixed offset per lane.  What it
        // fetches behind the last tile is the last whole one again (or, if there is none, pieces that exist) and is not used.
        const int whole = (kend - kbeg) / BK, rem = (kend - kbeg) % BK;
        const size_t pstep = (TP ? (size_t)BK * p.ldp : (size_t)BK) * sizeof(T), qstep = (TQ ? (size_t)BK * p.ldq : (size_t)BK) * sizeof(T);
        const char *pb = (const char*)P, *qb = (const char*)Q;
        int todo = whole;
        auto advance = [&]() {
            todo--;
            pb += todo > 0 ? pstep : 0;
            qb += todo > 0 ? qstep : 0;
        };
        if (whole == 0) {
#pragma unroll
            for (int j = 0; j < PN; j++)
                if (pk[j] >= rem) poff[j] = 0;
#pragma unroll
            for (int j = 0; j < QN; j++)
                if (qk[j] >= rem) qoff[j] = 0;
        }
        auto source = [&](int j) { return j < PN ? pb + poff[j < PN ? j : 0] : qb + qoff[j < PN ? 0 : j - PN]; };
        auto tail_source = [&](int j) {
            const char* src = j < PN ? (const char*)P + whole * pstep + poff[j < PN ? j : 0] : (const char*)Q + whole * qstep + qoff[j < PN ? 0 : j - PN];
            return (j < PN ? pk[j < PN ? j : 0] : qk[j < PN ? 0 : j - PN]) < rem ? src : (const char*)&zero_piece;
        };
        auto place1 = [&](int j, unsigned char* st) { return st + (j < PN ? 0 : SP::BYTES) + (wave + (j < PN ? j : j - PN) * NW) * 1024; };
        auto dma = [&](const char* src, int j, unsigned char* st) { __builtin_amdgcn_global_load_lds((glb_void*)src, (lds_void*)place1(j, st), 16, 0, 0); };
        f32x4 rg[STAGED ? PN + QN : 1];
        auto fetch = [&]() {  // a tile into registers
#pragma unroll
            for (int j = 0; j < PN + QN; j++) rg[STAGED ? j : 0] = *reinterpret_cast<const f32x4*>(source(j));
            advance();
        };
        auto put1 = [&](int j, unsigned char* st) { *reinterpret_cast<f32x4*>(place1(j, st) + lane * 16) = rg[STAGED ? j : 0]; };
        F fp[2][TRN], fq[2][TCN];
        if constexpr (STAGED) {
            if (rem) {
#pragma unroll
                for (int j = 0; j < PN + QN; j++) rg[STAGED ? j : 0] = *reinterpret_cast<const f32x4*>(tail_source(j));
            } else {
                fetch();
            }
#pragma unroll
            for (int j = 0; j < PN + QN; j++) put1(j, smem);
            fetch();
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < NS; i++) {
                if (i == 0 && rem) {
#pragma unroll
                    for (int j = 0; j < PN + QN; j++) dma(tail_source(j), j, smem);
                } else {
#pragma unroll
                    for (int j = 0; j < PN + QN; j++) dma(source(j), j, smem + i * STAGE);
                    advance();
                }
            }
            dma_wait_barrier<(NS - 1) * (PN + QN)>();
        }
#pragma unroll
        for (int j = 0; j < TCN; j++) fq[0][j] = qfrag(smem, j, 0);
#pragma unroll
        for (int i = 0; i < TRN; i++) fp[0][i] = pfrag(smem, i, 0);
        // one copy of the matrix instructions per place in LDS and no branch in it
        auto tile = [&](unsigned char* cur, unsigned char* nxt) {
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
                        for (int e = i * (PN + QN) / TRN; e < (i + 1) * (PN + QN) / TRN; e++) dma(source(e), e, cur);
                        if (i == TRN - 1) advance();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        if constexpr (NS == 2) {
            for (int kt = 0;;) {
                tile(smem, smem + STAGE);
                if (++kt >= nk) break;
                tile(smem + STAGE, smem);
                if (++kt >= nk) break;
            }
        } else {
            unsigned char *cur = smem, *nxt = smem + STAGE;
            for (int kt = 0; kt < nk; kt++) {
                tile(cur, nxt);
                cur = nxt;
                nxt = cur == smem + (NS - 1) * STAGE ? smem : cur + STAGE;
            }
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the last of them have landed before LDS is used again
    }

    // ---- epilogue: 16 rows of the wave's columns at a time through LDS rows of its own (two sets: the next rows are written while these
    // are worked on), then 8 adjacent columns per lane.  The residual of the next 16 rows is fetched meanwhile; a lane's columns stay the same.
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // the last matrix instructions have retired before their registers are read
    __syncthreads();                                     // every wave is done with the operand tiles
    float* ot = reinterpret_cast<float*>(smem) + wave * 2 * 16 * OS;
    const int i16 = lane & 15, q4 = lane >> 4;
    constexpr int LPR = WCOLS / 8, ITEMS = 16 * LPR / 64, STEP = 64 / LPR;  // lanes per row; rows between a lane's items
    static_assert(ITEMS >= 1 && 64 % LPR == 0, "a wave has 32, 64 or more columns");
    float* part = p.splits > 1 ? p.part + (size_t)split * p.R * p.C : nullptr;
    const bool use_res = FULL && p.res && p.vec && !part;
    const int rl = lane / LPR, cl = lane % LPR * 8, rfirst = r0 + wr * (BR / WR) + rl, c = c0 + wc * WCOLS + cl, n = min(8, p.C - c);
    float bias[8];
    load_bias<FULL>(p, c, bias);
    Frag<T> rn[ITEMS];
    auto fetch_res = [&](int i) {
#pragma unroll
        for (int it = 0; it < ITEMS; it++) {
            const int r = rfirst + i * 16 + it * STEP;
            if (r < p.R && n > 0) frag_load<T>(rn[it], (const T*)p.res + (size_t)r * p.ldr + c);
        }
    };
    auto put_rows = [&](auto row) {
        constexpr int i = decltype(row)::value;
#pragma unroll
        for (int j = 0; j < TCN; j++) *reinterpret_cast<f32x4*>(ot + (i & 1) * 16 * OS + i16 * OS + j * 16 + q4 * 4) = acc[i][j];
    };
    auto finish = [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (use_res) fetch_res(0);
        put_rows(std::integral_constant<int, 0>());
        static_for<TRN>([&](auto row) {
            constexpr int i = decltype(row)::value;
            __builtin_amdgcn_wave_barrier();
            f32x4 a[ITEMS], b[ITEMS];
            Frag<T> rv[ITEMS];
#pragma unroll
            for (int it = 0; it < ITEMS; it++) {
                const float* at = ot + (i & 1) * 16 * OS + (rl + it * STEP) * OS + cl;
                a[it] = *reinterpret_cast<const f32x4*>(at);
                b[it] = *reinterpret_cast<const f32x4*>(at + 4);
                rv[it] = rn[it];
            }
            if constexpr (i + 1 < TRN) {
                put_rows(std::integral_constant<int, i + 1>());
                if (use_res) fetch_res(i + 1);
            }
            __builtin_amdgcn_wave_barrier();
            if (p.vec) {
#pragma unroll
                for (int it = 0; it < ITEMS; it++) {
                    const int r = rfirst + i * 16 + it * STEP;
                    if (r < p.R && n > 0) {
                        float v[8] = {a[it][0], a[it][1], a[it][2], a[it][3], b[it][0], b[it][1], b[it][2], b[it][3]};
                        if (part) {
                            float* d = part + (size_t)r * p.C + c;
                            *reinterpret_cast<f32x4*>(d) = a[it];
                            *reinterpret_cast<f32x4*>(d + 4) = b[it];
                        } else {
                            epi8<T, ACT, FULL>(p, v, r, c, rv[it], bias);
                        }
                    }
                }
            } else {  // value by value, adjacent lanes on adjacent columns
#pragma unroll
                for (int it = 0; it < 16 * WCOLS / 64; it++) {
                    const int e = it * 64 + lane, y = e / WCOLS, x = e % WCOLS, r = r0 + wr * (BR / WR) + i * 16 + y, cc = c0 + wc * WCOLS + x;
                    const float z = ot[(i & 1) * 16 * OS + y * OS + x];
                    if (r < p.R && cc < p.C) {
                        if (part) part[(size_t)r * p.C + cc] = z;
                        else epi1<T, ACT, FULL>(p, z, r, cc);
                    }
                }
            }
        });
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

// MINW waves per SIMD: it bounds the registers, and with at most 256 of them hipcc keeps the accumulators where the matrix instructions read them (with
// more it moves them between the two register files in every K step)
template <typename T, int BR, int BC, int WR, int WC, int NS, int MINW> __global__ __launch_bounds__(WR* WC * 64, MINW) void linear_kernel(LinP p, int rtiles, int ctiles) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    linear_tile<T, false, false, BR, BC, WR, WC, NS, true>(p, rtiles, ctiles, blockIdx.x, smem);
}

// ---- few outputs: a block takes 32 x 32 of them, its four waves every fourth K step.  The fragments come straight from memory (the operands are
// small and shared through L2), all of a wave's loads for 4 steps in flight; the partial sums meet in LDS.  No k slices over blocks, so
// one launch.  20x1536x384 with GELU and pre: 4.7 us in bf16, 7.6 in fp32 (traced).  ALIGNED: rows of whole 16 bytes; otherwise value by value.
template <typename T, bool ALIGNED> __global__ __launch_bounds__(256) void linear_small_kernel(LinP p, int ctiles) {
    using F = typename Ops<T>::F;
    constexpr int E = 16 / (int)sizeof(T), KK = Ops<T>::KK, OS = 36;
    __shared__ float sm[4][32 * OS];
    const int rt = blockIdx.x / ctiles, r0 = rt * 32, c0 = (blockIdx.x - rt * ctiles) * 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q4 = lane >> 4;
    const T *ps[2], *qs[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        ps[i] = (const T*)p.p + (size_t)min(r0 + i * 16 + i16, p.R - 1) * p.ldp + q4 * E;
        qs[i] = (const T*)p.q + (size_t)min(c0 + i * 16 + i16, p.C - 1) * p.ldq + q4 * E;
    }
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](const T* src, int k) {  // E values from k + q4 E on; zero past the end
        F f = {};
        const int left = p.K - (k + q4 * E);
        if constexpr (ALIGNED) {
            if (left > 0) f = *reinterpret_cast<const F*>(src + k);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (e < left) f[e] = src[k + e];
        }
        return f;
    };
    constexpr int U = 4;
    const int steps = (p.K + KK - 1) / KK;
    for (int s = wave; s < steps; s += 4 * U) {
        F fp[U][2], fq[U][2];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < 2; i++) {  // steps past the end load zeros
                fp[u][i] = load(ps[i], (s + 4 * u) * KK);
                fq[u][i] = load(qs[i], (s + 4 * u) * KK);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) Ops<T>::mma(acc[i][j], fq[u][j], fp[u][i]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) *reinterpret_cast<f32x4*>(&sm[wave][(i * 16 + i16) * OS + j * 16 + q4 * 4]) = acc[i][j];
    __syncthreads();
    // adjacent lanes on adjacent columns: 8 rows at a time
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int y = it * 8 + (threadIdx.x >> 5), x = threadIdx.x & 31, r = r0 + y, c = c0 + x, o = y * OS + x;
        if (r >= p.R || c >= p.C) continue;
        const float z = (sm[0][o] + sm[1][o]) + (sm[2][o] + sm[3][o]);
        if (p.act == ACT_RELU) epi1<T, ACT_RELU, true>(p, z, r, c);
        else if (p.act == ACT_GELU) epi1<T, ACT_GELU, true>(p, z, r, c);
        else if (p.act == ACT_SILU) epi1<T, ACT_SILU, true>(p, z, r, c);
        else epi1<T, ACT_NONE, true>(p, z, r, c);
    }
}

// ---- operands whose rows do not lie on 16 bytes, copied to rows that do (zeros behind them): a thread moves 16 bytes
struct PackP {
    const void* src[2];
    void* dst[2];
    long long ld[2];
    long long n[2];  // 16-byte pieces; 0: nothing to do
    int K, per_row;  // values and pieces of a row
};
template <typename T> __device__ __forceinline__ void pack1(const T* src, T* dst, int left) {
    constexpr int E = 16 / (int)sizeof(T);
    unsigned w[4] = {0, 0, 0, 0};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (e < left) w[e] = __builtin_bit_cast(unsigned, src[e]);
    } else {  // whole words that hold at least one of the values, shifted into place
        const bool odd = ((uintptr_t)src & 2) != 0;
        const unsigned* q = reinterpret_cast<const unsigned*>((uintptr_t)src & ~(uintptr_t)3);
        unsigned v[5];
        const int have = min(left, E) + (odd ? 1 : 0);  // halves from q on
#pragma unroll
        for (int e = 0; e < 5; e++) v[e] = 2 * e < have ? q[e] : 0u;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w[e] = odd ? (v[e] >> 16) | (v[e + 1] << 16) : v[e];
            if (2 * e >= left) w[e] = 0;
            else if (2 * e + 1 >= left) w[e] &= 0xffffu;
        }
    }
    *reinterpret_cast<f32x4*>(dst) = f32x4{__builtin_bit_cast(float, w[0]), __builtin_bit_cast(float, w[1]), __builtin_bit_cast(float, w[2]), __builtin_bit_cast(float, w[3])};
}
template <typename T> __device__ __forceinline__ void linear_pack(const PackP& p, int blk) {
    constexpr int E = 16 / (int)sizeof(T);
    long long i = (long long)blk * 256 + threadIdx.x;
    int which = 0;
    if (i >= p.n[0]) {
        i -= p.n[0];
        which = 1;
    }
    if (i >= p.n[which]) return;
    const long long r = i / p.per_row;
    const int k = (int)(i - r * p.per_row) * E;
    pack1<T>((const T*)p.src[which] + r * p.ld[which] + k, (T*)p.dst[which] + i * E, p.K - k);
}
template <typename T> __global__ __launch_bounds__(256) void linear_pack_kernel(PackP p) { linear_pack<T>(p, blockIdx.x); }

// splits > 1: the partial products of a row's 8 columns (one column where rows are not stored as vectors: adjacent lanes on adjacent values),
// added in order, and the epilogue.  8 columns per thread whatever the alignment: 5000x100x300 backward 29 us in bf16 and 42 in fp32, now 20 and 26.
template <typename T, int ACT, bool FULL> __device__ __forceinline__ void linear_join(const LinP& p, int blk) {
    const long long i = (long long)blk * 256 + threadIdx.x;
    const size_t step = (size_t)p.R * p.C;
    if (p.vec) {
        const int cv = p.C / 8;
        if (i >= (long long)p.R * cv) return;
        const int r = (int)(i / cv), c = (int)(i - (long long)r * cv) * 8;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const float* s = p.part + (size_t)r * p.C + c;
#pragma unroll 4
        for (int k = 0; k < p.splits; k++) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(s + k * step), b = *reinterpret_cast<const f32x4*>(s + k * step + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] += a[e];
                v[4 + e] += b[e];
            }
        }
        Frag<T> rv;
        if (FULL && p.res) frag_load<T>(rv, (const T*)p.res + (size_t)r * p.ldr + c);
        float bias[8];
        load_bias<FULL>(p, c, bias);
        epi8<T, ACT, FULL>(p, v, r, c, rv, bias);
    } else {
        if (i >= (long long)step) return;
        const int r = (int)(i / p.C), c = (int)(i - (long long)r * p.C);
        float v = 0.f;
        const float* s = p.part + i;
#pragma unroll 8
        for (int k = 0; k < p.splits; k++) v += s[k * step];
        epi1<T, ACT, FULL>(p, v, r, c);
    }
}
inline long long join_blocks(const LinP& p) { return p.splits > 1 ? ((long long)p.R * (p.vec ? p.C / 8 : p.C) + 255) / 256 : 0; }
template <typename T, int ACT> __global__ __launch_bounds__(256) void linear_join_kernel(LinP p) { linear_join<T, ACT, true>(p, blockIdx.x); }

// ---- dz = dy act'(z), and the column sums of the unrounded dz.  A block takes `rows` rows of LP V columns: LP lanes (2^lg) side by side, the
// other 256 / LP threads share the rows, four of them in flight.  A thread adds at most 256 values in fp32: dz_rows sees to that for vectors of 8 columns; value by
// value (rows off 16 bytes) it has up to 8 times as many rows and goes on in fp64 after each 256.  One block of rows: its sums are db.  Bound by HBM:
// 6272x4096 bf16 with GELU 29 us = 5.3 TB/s.
struct DzP {
    const void *dy, *pre;
    long long ldy, ldpre;
    void* dz;       // [M][ldz], columns N .. ldz - 1 zero; NULL: only the sums
    float* part;    // [row blocks][N] (or db), or NULL
    int M, N, ldz, rows, cols, lg;  // cols: blocks of columns
};
template <typename T, int V, int ACT> __device__ __forceinline__ void linear_dz(const DzP& p, int blk, float* sm) {  // sm: 4 rows of 64 V
    const int by = blk / p.cols, bx = blk - by * p.cols, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lp = 1 << p.lg, cx = lane & (lp - 1);
    const int c = (bx * lp + cx) * V, rt = 256 >> p.lg, width = p.dz ? p.ldz : p.N;
    const long long row0 = (long long)by * p.rows, row1 = row0 + p.rows < p.M ? row0 + p.rows : p.M;
    float s[V];
#pragma unroll
    for (int j = 0; j < V; j++) s[j] = 0.f;
    if (c < width) {
        constexpr int U = 4;
        double before = 0.0;
        int added = 0;
        for (long long r0 = row0 + (wave << (6 - p.lg)) + (lane >> p.lg); r0 < row1; r0 += U * rt) {
            Frag<T> fd[V == 8 ? U : 1], fp[V == 8 && ACT != ACT_NONE ? U : 1];
            float d[U], z[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long r = r0 + u * rt;
                d[u] = 0.f;
                if (r < row1) {
                    if constexpr (V == 8) {
                        frag_load<T>(fd[u], (const T*)p.dy + r * p.ldy + c);
                        if constexpr (ACT != ACT_NONE) frag_load<T>(fp[u], (const T*)p.pre + r * p.ldpre + c);
                    } else if (c < p.N) {
                        d[u] = to_f32<T>(((const T*)p.dy)[r * p.ldy + c]);
                        if constexpr (ACT != ACT_NONE) z[u] = to_f32<T>(((const T*)p.pre)[r * p.ldpre + c]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long r = r0 + u * rt;
                if (r >= row1) continue;
                if constexpr (V == 8) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        v[j] = frag_get<T>(fd[u], j);
                        if constexpr (ACT != ACT_NONE) v[j] *= act_slope<T, ACT>(frag_get<T>(fp[u], j));
                        s[j] += v[j];
                    }
                    if (p.dz) {
#pragma unroll
                        for (int j = 0; j < 8; j++) frag_set<T>(fd[u], j, v[j]);
                        frag_store<T>(fd[u], (T*)p.dz + r * p.ldz + c);
                    }
                } else {
                    if constexpr (ACT != ACT_NONE)
                        if (c < p.N) d[u] *= act_slope<T, ACT>(z[u]);
                    if (p.dz) ((T*)p.dz)[r * p.ldz + c] = from_f32<T>(d[u]);
                    s[0] += d[u];
                }
            }
            if constexpr (V == 1)
                if ((added += U) == 256) {
                    before += (double)s[0];
                    s[0] = 0.f;
                    added = 0;
                }
        }
        if constexpr (V == 1) s[0] = (float)(before + (double)s[0]);
    }
    if (!p.part) return;
#pragma unroll
    for (int j = 0; j < V; j++)
        for (int o = lp; o < 64; o <<= 1) s[j] += __shfl_xor(s[j], o, 64);
    const int W = lp * V;
    if (lane < lp) {
#pragma unroll
        for (int j = 0; j < V; j++) sm[wave * W + cx * V + j] = s[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < W; i += 256) {
        const int col = bx * W + i;
        if (col < p.N) p.part[(size_t)by * p.N + col] = (float)(((double)sm[i] + (double)sm[W + i]) + ((double)sm[2 * W + i] + (double)sm[3 * W + i]));
    }
}
// what the products need first, in one launch: the first nd blocks write dz, the others pack x and w
template <typename T, int V, int ACT> __global__ __launch_bounds__(256) void linear_dz_kernel(DzP p, PackP pp, int nd) {
    __shared__ float sm[4 * 64 * V];
    if ((int)blockIdx.x < nd) linear_dz<T, V, ACT>(p, blockIdx.x, sm);
    else linear_pack<T>(pp, (int)blockIdx.x - nd);
}
__device__ __forceinline__ void linear_db(const float* part, float* db, int chunks, int N, int blk) {
    // 16 lanes x 16 columns: 16 strides of the chunks, joined in LDS in fp64
    __shared__ double sm[16][17];
    const int cx = threadIdx.x & 15, y = threadIdx.x >> 4, c = blk * 16 + cx;
    double s = 0.0;
    if (c < N)
#pragma unroll 8
        for (int k = y; k < chunks; k += 16) s += (double)part[(size_t)k * N + c];
    sm[y][cx] = s;
    __syncthreads();
    if (y == 0 && c < N) {
        for (int k = 1; k < 16; k++) s += sm[k][cx];
        db[c] = (float)s;
    }
}

// ---- the products of the backward in one launch: the blocks of dW, those of dx and, without an activation, those of the column sums of dy.
// Tiles of TL x TL, two 128 x 128 blocks per CU; one launch fills the chip where dW (few tiles, long k) or dx alone would not, and the tails overlap.
struct BwdP {
    LinP w, x;
    int wr, wc, xr, xc;           // tiles
    int n0, n1;                   // blocks of the first and of the first two segments (multiples of 8, so that block index modulo 8 stays the XCD)
    int w_first;                  // the segment with the longer blocks comes first
    DzP s;
};
template <typename T, int TL, int SV> __global__ __launch_bounds__(256, 2) void linear_bwd_kernel(BwdP p) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int id = blockIdx.x;
    if (id >= p.n1) {
        linear_dz<T, SV, ACT_NONE>(p.s, id - p.n1, reinterpret_cast<float*>(smem));
        return;
    }
    const bool first = id < p.n0;
    const int at = first ? id : id - p.n0;
    if (first == (p.w_first != 0)) {
        if (at < p.wr * p.wc * p.w.splits) linear_tile<T, true, true, TL, TL, 2, 2, 2, false>(p.w, p.wr, p.wc, at, smem);
    } else {
        if (at < p.xr * p.xc * p.x.splits) linear_tile<T, false, true, TL, TL, 2, 2, 2, false>(p.x, p.xr, p.xc, at, smem);
    }
}
// what remains: the joins of dW and dx, and db from the column sums
template <typename T> __global__ __launch_bounds__(256) void linear_bwd_join_kernel(LinP w, LinP x, int nw, int nx, const float* sums, float* db, int chunks, int N) {
    const int id = blockIdx.x;
    if (id < nw) linear_join<T, ACT_NONE, false>(w, id);
    else if (id < nw + nx) linear_join<T, ACT_NONE, false>(x, id - nw);
    else linear_db(sums, db, chunks, N, id - nw - nx);
}

// ================================================== host ==================================================
inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

constexpr int TILE = 128;
inline int up(int a, int b) { return (a + b - 1) / b; }

void set_split(LinP& p, int s, int bk) {
    const int nk = up(p.K, bk), per = up(nk, s);
    p.splits = up(nk, per);
    p.kper = per * bk;
}

template <typename K> int raise_lds(K kern, size_t lds, std::atomic<bool>* set) {
    int dev = 0;
    (void)hipGetDevice(&dev);
    dev &= 63;
    if (!set[dev].load(std::memory_order_acquire)) {
        const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        DIG_CHECK(e == hipSuccess, DIG_ELAUNCH, "linear_act: cannot raise dynamic LDS to %zu: %s", lds, hipGetErrorString(e));
        set[dev].store(true, std::memory_order_release);
    }
    return DIG_OK;
}
template <int BR, int BC, int NW, int WC, int NS> constexpr size_t lds_of() {
    constexpr size_t stages = (size_t)NS * (BR + BC) * KB, rows = (size_t)NW * 2 * 16 * (BC / WC + 4) * 4;
    return stages > rows ? stages : rows;
}

// ---- forward
template <typename T, int BR, int BC, int WR, int WC, int NS, int MINW> int fwd_launch(const LinP& p, hipStream_t st) {
    constexpr size_t lds = lds_of<BR, BC, WR * WC, WC, NS>();
    auto kern = linear_kernel<T, BR, BC, WR, WC, NS, MINW>;
    if constexpr (lds > 64 * 1024) {
        static std::atomic<bool> set[64];
        const int rc = raise_lds(kern, lds, set);
        if (rc != DIG_OK) return rc;
    }
    const int rt = up(p.R, BR), ct = up(p.C, BC);
    hipLaunchKernelGGL(kern, dim3((unsigned)(rt * ct * p.splits)), dim3(WR * WC * 64), lds, st, p, rt, ct);
    if (p.splits > 1) {
        const dim3 grid((unsigned)join_blocks(p));
        switch (p.act) {
            case ACT_RELU: hipLaunchKernelGGL((linear_join_kernel<T, ACT_RELU>), grid, dim3(256), 0, st, p); break;
            case ACT_GELU: hipLaunchKernelGGL((linear_join_kernel<T, ACT_GELU>), grid, dim3(256), 0, st, p); break;
            case ACT_SILU: hipLaunchKernelGGL((linear_join_kernel<T, ACT_SILU>), grid, dim3(256), 0, st, p); break;
            default: hipLaunchKernelGGL((linear_join_kernel<T, ACT_NONE>), grid, dim3(256), 0, st, p); break;
        }
    }
    DIG_LAUNCH_CHECK("linear_act");
    return DIG_OK;
}

enum { TILE_SMALL = 0, TILE_64 = 1, TILE_128 = 2, TILE_192 = 3, TILE_256 = 4, TILE_64_SHORT = 5 };
// Tile and k slices of the forward: the least estimated time.  A block of a tile costs fill + k tiles * step us while its CU holds as many
// blocks as fit (slots in all).  Measured, GELU with pre kept (last three: not kept), us, in brackets what is taken; "short" are 64 x 64 tiles with two
// stages in LDS instead of four, four blocks per CU instead of two: ahead for many tiles of few k, behind (43 to 41 and 477 to 466) otherwise:
//   M x N x K              64     128   192x128   256 |  fp32: 64   128   192x128   256  short
//   1024 x 1024 x 1024   [7.8]   13.7    18.0    32.6 |     [25]    73       109    276
//   4096 x 1024 x 1024    20.6  [17.8]   22.4    35.8 |      80    [75]      111    268
//   6912 x 1536 x  384    34.6   26.4   [24.1]   27.5 |      97    112        95    121   [90]
//   6912 x  384 x 1536   [20.6]  24.0    28.8    43.7 |     [86]   104       155    389
//   6272 x 4096 x 1024     104    77      76     [74] |     465   [475]      518    545
//   8192 x 4096 x 4096     406   254     261    [223] |
//   9409 x  408 x  168                                |      32     41        38          [27]
//  30001 x   96 x   48                                |    16.9   18.9      25.3        [13.5]
//  12288 x 1000 x  800                                |     184             [174]
// 256 x 256 is not built for fp32: it won nowhere.  Few outputs take linear_small_kernel (20x1536x384, traced: 4.7 against 6.4; fp32 7.6 against 13.4); few
// outputs of a long sum are cut into k slices of 64 x 64 tiles, whose join costs a launch and the partial sums' bytes (256x256x8192: 11.8 against 25.6 uncut).
int fwd_plan(int M, int N, int K, int dtype, int& splits) {
    struct Cost {
        int br, bc, slots;
        double fill, step, alone;  // alone: a step where no CU holds two blocks
    };
    static const Cost cost16[] = {{64, 64, 512, 4.5, 0.445, 0.445}, {128, 128, 512, 7.4, 1.15, 1.15}, {192, 128, 512, 14.0, 1.5, 1.5}, {256, 256, 256, 19.2, 1.61, 1.61}};
    static const Cost cost32[] = {{64, 64, 512, 5.5, 1.0, 0.57}, {128, 128, 512, 16.0, 3.8, 1.83}, {192, 128, 512, 19.7, 6.2, 2.82}, {64, 64, 1024, 10.0, 1.57, 1.57}};
    const bool f32 = dtype != DIG_BF16;
    const int nk = up(K, f32 ? 32 : 64);
    splits = 1;
    const long long small = (long long)up(M, 32) * up(N, 32);
    const bool odd = K % (f32 ? 4 : 8) != 0;  // read value by value by linear_small_kernel, packed for the others: 501x333x777 in bf16 24 against 14 us
    double best = small <= 512 ? (3.0 + (odd ? 0.026 * K : up(K, f32 ? 256 : 512) * (f32 ? 1.5 : 1.2))) * (small <= 256 ? 1.0 : 1.6) : 1e30;
    int tile = TILE_SMALL;
    for (int i = 0; i < 4; i++) {
        const Cost& c = f32 ? cost32[i] : cost16[i];
        const double tiles = (double)up(M, c.br) * up(N, c.bc), full = tiles / c.slots;
        if (f32 && i == 3 && (tiles <= 512.0 || nk > 12)) break;
        double rounds = full <= 1.0 ? 1.0 : full + 0.4;
        if (full > 1.0 && rounds > (double)(long long)full + 1.0) rounds = (double)(long long)full + 1.0;
        const double t = rounds * (c.fill + nk * (tiles <= 256.0 ? c.alone : c.step)) + (odd ? 4.0 : 0.0);
        if (t < best) {
            best = t;
            tile = f32 && i == 3 ? TILE_64_SHORT : TILE_64 + i;
        }
    }
    const long long t64 = (long long)up(M, 64) * up(N, 64);
    if (t64 <= 128 && nk >= 16) {
        int n = (int)(512 / t64);
        if (n > nk / 8) n = nk / 8;
        if (n > 64) n = 64;
        n = up(nk, up(nk, n));
        if (n > 1 && 4.5 + up(nk, n) * (f32 ? 0.9 : 0.445) + 6.0 + 8.0 * n * M * N / 4.5e6 < best) {
            splits = n;
            tile = TILE_64;
        }
    }
    return tile;
}

// byte offsets inside a tile are 31 bits: up to 256 rows of a k-adjacent operand, the tile's k rows of the others
bool offsets_ok(long long ld, bool k_adjacent, int esize) { return ld * (k_adjacent ? 256 : KB / esize) * esize < (1ll << 31); }

// an operand of 16-byte rows, or its packed copy's place; false: it has to be packed and there is no place for it
struct Operand {
    const void* p;
    long long ld;
};
template <typename T> bool operand(const void* src, long long ld, bool k_adjacent, int rows, int K, void* pack, PackP& pp, int slot, Operand& o) {
    const int E = 16 / (int)sizeof(T);
    o = {src, ld};
    if (K % E == 0 && ld % E == 0 && al16(src) && offsets_ok(ld, k_adjacent, (int)sizeof(T))) return true;
    if (!pack || !al16(pack)) return false;
    pp.src[slot] = src;
    pp.dst[slot] = pack;
    pp.ld[slot] = ld;
    pp.K = K;
    pp.per_row = up(K, E);
    pp.n[slot] = (long long)rows * pp.per_row;
    o = {pack, (long long)pp.per_row * E};
    return true;
}
long long pack_blocks(const PackP& pp) { return (pp.n[0] + pp.n[1] + 255) / 256; }

template <typename T> int fwd(const dig_linear_act_args* a, hipStream_t st) {
    const int E = 16 / (int)sizeof(T);
    LinP p{};
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
    int splits;
    const int tile = fwd_plan(a->M, a->N, a->K, a->dtype, splits);
    if (tile == TILE_SMALL) {
        p.p = a->x;
        p.q = a->w;
        p.ldp = a->ldx;
        p.ldq = a->ldw;
        const int ct = up(p.C, 32);
        const dim3 grid((unsigned)(up(p.R, 32) * ct));
        if (a->K % E == 0 && a->ldx % E == 0 && a->ldw % E == 0 && al16(a->x) && al16(a->w)) hipLaunchKernelGGL((linear_small_kernel<T, true>), grid, dim3(256), 0, st, p, ct);
        else hipLaunchKernelGGL((linear_small_kernel<T, false>), grid, dim3(256), 0, st, p, ct);
        DIG_LAUNCH_CHECK("linear_act");
        return DIG_OK;
    }
    PackP pp{};
    Operand x, w;
    DIG_CHECK(operand<T>(a->x, a->ldx, true, a->M, a->K, a->xpack, pp, 0, x) && operand<T>(a->w, a->ldw, true, a->N, a->K, a->wpack, pp, 1, w), DIG_EALIGN,
              "linear_act: rows that do not lie on 16 bytes need xpack / wpack");
    DIG_CHECK(grid_fits(pack_blocks(pp), 256), DIG_EINVAL, "linear_act: too many blocks");
    if (pack_blocks(pp)) hipLaunchKernelGGL((linear_pack_kernel<T>), dim3((unsigned)pack_blocks(pp)), dim3(256), 0, st, pp);
    p.p = x.p;
    p.q = w.p;
    p.ldp = x.ld;
    p.ldq = w.ld;
    set_split(p, splits, KB / (int)sizeof(T));
    switch (tile) {
        case TILE_64: return fwd_launch<T, 64, 64, 2, 2, 4, 2>(p, st);
        case TILE_64_SHORT:
            if constexpr (sizeof(T) == 4) return fwd_launch<T, 64, 64, 2, 2, 2, 4>(p, st);
        case TILE_192: return fwd_launch<T, 192, 128, 2, 2, 2, 2>(p, st);
        case TILE_256:
            if constexpr (sizeof(T) == 2) return fwd_launch<T, 256, 256, 2, 4, 2, 2>(p, st);
        default: return fwd_launch<T, 128, 128, 2, 2, 2, 2>(p, st);
    }
}

// ---- backward
struct BwdPlan {
    int tile, sx, sw;  // tile 64 or 128, k slices of dx and of dW
};
// when n1 blocks of length b1 and then n2 of length b2 <= b1 are done, over `slots` that take the next block as they become free
double makespan(double n1, double b1, double n2, double b2, double slots) {
    const double q = (double)(long long)(n1 / slots), rem = n1 - q * slots, t0 = q * b1, t1 = rem > 0 ? t0 + b1 : t0;
    if (n2 <= 0) return t1;
    double best = 1e30;
    for (int e = 0; e < 2; e++) {
        const double base = e ? t1 : t0;
        double j = (double)(long long)(((q * b1 * slots + rem * b1 + n2 * b2) / slots - base) / b2) - 1.0;
        if (j < 1.0) j = 1.0;
        for (int s = 0; s < 4; s++, j += 1.0) {
            const double t = base + j * b2 + 1e-9;
            if (t < t1) continue;
            if ((slots - rem) * (double)(long long)((t - t0) / b2) + rem * (double)(long long)((t - t1) / b2) >= n2) {
                if (t < best) best = t;
                break;
            }
        }
    }
    return best < 1e30 ? best : t1 + (n2 / slots + 1.0) * b2;
}
// Rows of a block of linear_dz (a function of M and N alone: the workspace depends on it): about 1024 blocks in all, at least 4 rows and at most
// 256 per thread, one block of rows where that makes at most 32 per thread (8 times as many where rows of 8 k values are misaligned).  4 rows in flight and narrow rows side by side in a wave:
// 15722 x 64 in fp32 took 24.6 us with 64 lanes across the columns whatever N is and one row in flight.
int lanes_log(int width, int V) {
    int lg = 0;
    while (lg < 6 && (V << lg) < width) lg++;
    return lg;
}
int dz_rows(int M, int N) {
    const int V = N % 8 == 0 ? 8 : 1, lg = lanes_log(N, V), rt = 256 >> lg;
    if (M <= 32 * rt) return M;
    const int cols = up(N, V << lg), want = cols < 1024 ? 1024 / cols : 1;
    int rows = up(M, want);
    if (rows < 4 * rt) rows = 4 * rt;
    if (rows > 256 * rt) rows = 256 * rt;
    return rows;
}
int dz_chunks(int M, int N) { return up(M, dz_rows(M, N)); }
// The least estimated time of one launch of both products.  A block costs fill + its k tiles * step us (measured on dx of 6912x1536x384 and
// 6272x1024x4096 in bf16: tile 64 28 / 119 us, tile 128 23 / 82 us; fp32 steps are the matrix units' own time); what is split is written and read again as fp32.
BwdPlan bwd_search(int M, int N, int K, int dtype, bool dx) {
    static const int cuts[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32, 48, 64};
    const bool f32 = dtype != DIG_BF16;
    const int bk = f32 ? 32 : 64, nkx = up(N, bk), nkw = up(M, bk);
    BwdPlan plan{128, 1, 1};
    double best = 1e30;
    const bool one_chunk = dz_chunks(M, N) == 1;
    for (int tile = 64; tile <= 128; tile += 64) {
        const double fill = tile == 64 ? 2.5 : f32 ? 6.0 : 11.0, step = tile == 64 ? (f32 ? 0.95 : 0.58) : (f32 ? 3.6 : 1.1);
        const double tx = dx ? (double)up(M, tile) * up(K, tile) : 0.0, tw = (double)up(N, tile) * up(K, tile);
        for (int a : cuts) {
            if (a > 1 && (!dx || nkx < 4 * a || tx * a > 2048)) break;
            for (int b : cuts) {
                if (b > 1 && (nkw < 4 * b || tw * b > 2048)) break;
                const double st = tx * a + tw * b <= 256.0 ? 0.8 * step : step;  // a block alone on its CU
                const double bx = fill + up(nkx, a) * st, bw = fill + up(nkw, b) * st;
                double t = !dx || bw >= bx ? makespan(tw * b, bw, tx * a, bx, 512.0) : makespan(tx * a, bx, tw * b, bw, 512.0);
                if (a > 1) t += 8.0 * a * M * K / 4.5e6;
                if (b > 1) t += 8.0 * b * N * K / 4.5e6;
                if ((a > 1 || b > 1) && one_chunk) t += 4.0;  // db needs no join: this one is a launch of its own
                if (t < best - 1e-9) {
                    best = t;
                    plan = {tile, a, b};
                }
            }
        }
    }
    plan.sx = up(nkx, up(nkx, plan.sx));
    plan.sw = up(nkw, up(nkw, plan.sw));
    return plan;
}
// the search takes a few us: a thread remembers its last shapes' plans
BwdPlan bwd_plan(int M, int N, int K, int dtype, bool dx) {
    struct Entry {
        int M, N, K, key;
        BwdPlan plan;
    };
    static thread_local Entry seen[64];
    const int key = 1 + dtype * 2 + (dx ? 1 : 0);
    Entry& e = seen[((unsigned)M * 31u + (unsigned)N * 17u + (unsigned)K * 7u + (unsigned)key) & 63];
    if (e.key != key || e.M != M || e.N != N || e.K != K) e = {M, N, K, key, bwd_search(M, N, K, dtype, dx)};
    return e.plan;
}

// fewer than 2^22 tiles of 128 x 128: the grids of 64 x 64 tiles hold fewer than 2^32 threads, and block numbers fit an int
bool shape_ok(int M, int N, int K) {
    return M > 0 && N > 0 && K > 0 && M <= (1 << 30) && N <= (1 << 20) && K <= (1 << 20) && (long long)((M + TILE - 1) / TILE) * ((N + TILE - 1) / TILE) < (1 << 22) &&
           (long long)((M + TILE - 1) / TILE) * ((K + TILE - 1) / TILE) < (1 << 22);
}

template <typename T, int ACT> void dz_launch(const DzP& d, const PackP& pp, int nd, bool vec, hipStream_t st) {
    const dim3 grid((unsigned)(nd + pack_blocks(pp)));
    if (vec) hipLaunchKernelGGL((linear_dz_kernel<T, 8, ACT>), grid, dim3(256), 0, st, d, pp, nd);
    else hipLaunchKernelGGL((linear_dz_kernel<T, 1, ACT>), grid, dim3(256), 0, st, d, pp, nd);
}

long long sum_floats(int M, int N) {
    const long long chunks = dz_chunks(M, N);
    return chunks > 1 ? (chunks * N + 3) / 4 * 4 : 0;
}
long long part_floats(const BwdPlan& q, int M, int N, int K, bool dx, long long& dx_floats) {
    dx_floats = dx && q.sx > 1 ? ((long long)q.sx * M * K + 3) / 4 * 4 : 0;
    return dx_floats + (q.sw > 1 ? (long long)q.sw * N * K : 0);
}

template <typename T> int bwd(const dig_linear_act_bwd_args* a, hipStream_t st) {
    const int E = 16 / (int)sizeof(T), es = (int)sizeof(T), M = a->M, N = a->N, K = a->K, ldz = up(N, 8) * 8;
    const int chunks = dz_chunks(M, N);
    float* sums = a->ws;  // column sums of row blocks, then the partial products of dx and dW
    float* part = a->ws + sum_floats(M, N);
    PackP pp{};
    Operand x, w{};
    DIG_CHECK(operand<T>(a->x, a->ldx, false, M, K, a->xpack, pp, 0, x) && (!a->dx || operand<T>(a->w, a->ldw, false, N, K, a->wpack, pp, 1, w)), DIG_EALIGN,
              "linear_act_bwd: rows that do not lie on 16 bytes need xpack / wpack");
    const Operand z = a->dz ? Operand{a->dz, ldz} : Operand{a->dy, a->ldy};
    DIG_CHECK(z.ld % E == 0 && al16(z.p) && (a->dz || N % E == 0) && offsets_ok(z.ld, true, es), DIG_EALIGN, "linear_act_bwd: rows of dy that do not lie on 16 bytes need dz");
    const bool dvec = N % 8 == 0 && a->ldy % 8 == 0 && al16(a->dy) && (a->act == ACT_NONE || (a->ldpre % 8 == 0 && al16(a->pre)));
    const int width = a->dz ? ldz : N, lg = lanes_log(width, dvec ? 8 : 1), dcols = up(width, (dvec ? 8 : 1) << lg);
    const DzP d{a->dy, a->pre, a->ldy, a->ldpre, a->dz, !a->db ? nullptr : chunks == 1 ? a->db : sums, M, N, ldz, dz_rows(M, N), dcols, lg};
    const BwdPlan plan = bwd_plan(M, N, K, a->dtype, a->dx != nullptr);
    long long xf;
    (void)part_floats(plan, M, N, K, a->dx != nullptr, xf);
    BwdP p{};
    p.w.p = p.x.p = z.p;  // dW[n][k] = sum_m dz[m][n] x[m][k],  dx[m][k] = sum_n dz[m][n] W[n][k]
    p.w.ldp = p.x.ldp = z.ld;
    p.w.q = x.p;
    p.w.ldq = x.ld;
    p.x.q = w.p;
    p.x.ldq = w.ld;
    p.w.R = N;
    p.w.rpad = up(N, E) * E;
    p.x.R = M;
    p.w.C = p.x.C = K;
    p.w.cpad = p.x.cpad = up(K, E) * E;
    p.w.K = M;
    p.x.K = N;
    p.w.out = a->dw;
    p.x.out = a->dx;
    p.w.ldo = p.x.ldo = K;
    p.w.out_f32 = a->dw_f32;
    p.w.vec = K % 8 == 0 && al16(a->dw);
    p.x.vec = K % 8 == 0 && al16(a->dx);
    p.x.part = part;
    p.w.part = part + xf;
    set_split(p.w, plan.sw, KB / es);
    set_split(p.x, plan.sx, KB / es);
    p.wr = up(N, plan.tile);
    p.wc = p.xc = up(K, plan.tile);
    p.xr = a->dx ? up(M, plan.tile) : 0;
    p.w_first = !a->dx || p.w.kper >= p.x.kper;
    const int nw = up(p.wr * p.wc * p.w.splits, 8) * 8, nx = up(p.xr * p.xc * p.x.splits, 8) * 8;
    p.n0 = p.w_first ? nw : nx;
    p.n1 = nw + nx;
    const bool sum_here = a->db && !a->dz;
    p.s = d;
    const dim3 grid((unsigned)(p.n1 + (sum_here ? dcols * chunks : 0)));
    const int nd = a->dz ? dcols * chunks : 0;
    DIG_CHECK(grid_fits(nd + pack_blocks(pp), 256) && grid_fits(grid.x, 256), DIG_EINVAL, "linear_act_bwd: too many blocks");
    if (nd + pack_blocks(pp)) {
        switch (a->dz ? a->act : ACT_NONE) {
            case ACT_RELU: dz_launch<T, ACT_RELU>(d, pp, nd, dvec, st); break;
            case ACT_GELU: dz_launch<T, ACT_GELU>(d, pp, nd, dvec, st); break;
            case ACT_SILU: dz_launch<T, ACT_SILU>(d, pp, nd, dvec, st); break;
            default: dz_launch<T, ACT_NONE>(d, pp, nd, dvec, st); break;
        }
    }
    constexpr size_t lds = lds_of<128, 128, 4, 2, 2>(), lds64 = lds_of<64, 64, 4, 2, 2>();
    static_assert(lds <= 64 * 1024, "no attribute needed");
    if (plan.tile == 128) {
        if (sum_here && dvec) hipLaunchKernelGGL((linear_bwd_kernel<T, 128, 8>), grid, dim3(256), lds, st, p);
        else hipLaunchKernelGGL((linear_bwd_kernel<T, 128, 1>), grid, dim3(256), lds, st, p);
    } else {
        if (sum_here && dvec) hipLaunchKernelGGL((linear_bwd_kernel<T, 64, 8>), grid, dim3(256), lds64, st, p);
        else hipLaunchKernelGGL((linear_bwd_kernel<T, 64, 1>), grid, dim3(256), lds64, st, p);
    }
    const int jw = (int)join_blocks(p.w), jx = a->dx ? (int)join_blocks(p.x) : 0, jd = a->db && chunks > 1 ? up(N, 16) : 0;
    if (jw + jx + jd) hipLaunchKernelGGL((linear_bwd_join_kernel<T>), dim3((unsigned)(jw + jx + jd)), dim3(256), 0, st, p.w, p.x, jw, jx, sums, a->db, chunks, N);
    DIG_LAUNCH_CHECK("linear_act_bwd");
    return DIG_OK;
}

}  // namespace

extern "C" int dig_linear_act_ws(int M, int N, int K, int dtype) {
    if (!shape_ok(M, N, K)) return DIG_EINVAL;
    int s;
    (void)fwd_plan(M, N, K, dtype, s);
    return s > 1 ? (int)((long long)s * M * N) : 0;
}
extern "C" int dig_linear_act_bwd_ws(int M, int N, int K, int dtype, int dx) {
    if (!shape_ok(M, N, K) || !shape_ok(N, K, 1)) return DIG_EINVAL;
    long long xf;
    const long long n = sum_floats(M, N) + part_floats(bwd_plan(M, N, K, dtype, dx != 0), M, N, K, dx != 0, xf);
    return n < (1ll << 31) ? (int)n : DIG_EINVAL;
}

extern "C" int dig_linear_act(const dig_linear_act_args* a, void* stream) {
    DIG_CHECK(a && a->x && a->w && a->out, DIG_EINVAL, "linear_act: null pointer");
    DIG_CHECK(shape_ok(a->M, a->N, a->K), DIG_EINVAL, "linear_act: bad shape M=%d N=%d K=%d", a->M, a->N, a->K);
    DIG_CHECK(a->act >= 0 && a->act <= 3, DIG_EINVAL, "linear_act: act %d", a->act);
    DIG_CHECK(a->dtype == DIG_BF16 || a->dtype == DIG_F32, DIG_EINVAL, "linear_act: dtype %d", a->dtype);
    DIG_CHECK(a->ldx >= 0 && a->ldw >= 0 && (!a->res || a->ldr >= 0), DIG_EINVAL, "linear_act: negative pitch");
    DIG_CHECK((a->ws && al16(a->ws)) || dig_linear_act_ws(a->M, a->N, a->K, a->dtype) == 0, DIG_EINVAL, "linear_act: this shape needs a workspace, on 16 bytes");
    return a->dtype == DIG_BF16 ? fwd<bf16>(a, (hipStream_t)stream) : fwd<float>(a, (hipStream_t)stream);
}

extern "C" int dig_linear_act_bwd(const dig_linear_act_bwd_args* a, void* stream) {
    DIG_CHECK(a && a->x && a->w && a->dy && a->dw, DIG_EINVAL, "linear_act_bwd: null pointer");
    DIG_CHECK(shape_ok(a->M, a->N, a->K) && shape_ok(a->N, a->K, 1), DIG_EINVAL, "linear_act_bwd: bad shape M=%d N=%d K=%d", a->M, a->N, a->K);
    DIG_CHECK(a->act >= 0 && a->act <= 3, DIG_EINVAL, "linear_act_bwd: act %d", a->act);
    DIG_CHECK(a->dtype == DIG_BF16 || a->dtype == DIG_F32, DIG_EINVAL, "linear_act_bwd: dtype %d", a->dtype);
    DIG_CHECK(a->act == ACT_NONE || (a->pre && a->dz), DIG_EINVAL, "linear_act_bwd: an activation needs pre and dz");
    DIG_CHECK(a->ldx >= 0 && a->ldw >= 0 && a->ldy >= 0 && (a->act == ACT_NONE || a->ldpre >= 0), DIG_EINVAL, "linear_act_bwd: negative pitch");
    const int need = dig_linear_act_bwd_ws(a->M, a->N, a->K, a->dtype, a->dx != nullptr);
    DIG_CHECK(need >= 0 && (need == 0 || a->ws), DIG_EINVAL, "linear_act_bwd: this shape needs a workspace");
    DIG_CHECK(al16(a->ws) && al16(a->dz), DIG_EINVAL, "linear_act_bwd: ws and dz have to lie on 16 bytes");
    return a->dtype == DIG_BF16 ? bwd<bf16>(a, (hipStream_t)stream) : bwd<float>(a, (hipStream_t)stream);
}
