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

template <bool FULL> __device__ __forceinline__ void load_bias(const LinP& p, int c, float (&bias)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) bias[j] = FULL && p.bias && c + j < p.C ? p.bias[c + j] : 0.f;
}

// 8 columns of the epilogue from column c of row r: n of them exist.  FULL: bias, pre, act and res; otherwise only the store.  rv: the
// residual's vector, if p.vec
template <typename T, int ACT, bool FULL> __device__ __forceinline__ void epi8(const LinP& p, float (&v)[8], int r, int c, int n, const Frag<T>& rv, const float (&bias)[8]) {
    const size_t o = (size_t)r * p.ldo + c;
    if (p.vec) {  // n is 8
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
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (j < n) {
            float z = v[j];
            if constexpr (FULL) {
                z += bias[j];
                if (p.pre) ((T*)p.pre)[o + j] = from_f32<T>(z);
                z = act_val<T, ACT>(z);
                if (p.res) z += to_f32<T>(((const T*)p.res)[(size_t)r * p.ldr + c + j]);
            }
            if (p.out_f32) ((float*)p.out)[o + j] = z;
            else ((T*)p.out)[o + j] = from_f32<T>(z);
        }
    }
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
#pragma unroll
            for (int it = 0; it < ITEMS; it++) {
                const int r = rfirst + i * 16 + it * STEP;
                if (r < p.R && n > 0) {
                    float v[8] = {a[it][0], a[it][1], a[it][2], a[it][3], b[it][0], b[it][1], b[it][2], b[it][3]};
                    if (part) {
                        float* d = part + (size_t)r * p.C + c;
                        if (n == 8 && p.C % 4 == 0) {
                            *reinterpret_cast<f32x4*>(d) = a[it];
                            *reinterpret_cast<f32x4*>(d + 4) = b[it];
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (e < n) d[e] = v[e];
                        }
                    } else {
                        epi8<T, ACT, FULL>(p, v, r, c, n, rv[it], bias);
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
template <typename T, int BR, int BC, int WR, int WC, int NS, int MINW, bool ALIGNED> __global__ __launch_bounds__(WR* WC * 64, MINW) void linear_kernel(LinP p, int rtiles, int ctiles) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    linear_tile<T, false, false, BR, BC, WR, WC, NS, ALIGNED, true>(p, rtiles, ctiles, blockIdx.x, smem);
}

// splits > 1: the partial products of a row's 8 columns, added in order, and the epilogue
template <typename T, int ACT, bool FULL> __device__ __forceinline__ void linear_join(const LinP& p, int blk) {
    const int cv = (p.C + 7) / 8;
    const long long i = (long long)blk * 256 + threadIdx.x;
    if (i >= (long long)p.R * cv) return;
    const int r = (int)(i / cv), c = (int)(i - (long long)r * cv) * 8, n = min(8, p.C - c);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const float* s = p.part + (size_t)r * p.C + c;
    const size_t step = (size_t)p.R * p.C;
    if (n == 8 && p.C % 4 == 0) {
#pragma unroll 4
        for (int k = 0; k < p.splits; k++) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(s + k * step), b = *reinterpret_cast<const f32x4*>(s + k * step + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] += a[e];
                v[4 + e] += b[e];
            }
        }
    } else {
        for (int k = 0; k < p.splits; k++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < n) v[e] += s[k * step + e];
    }
    Frag<T> rv;
    if (FULL && p.res && p.vec) frag_load<T>(rv, (const T*)p.res + (size_t)r * p.ldr + c);
    float bias[8];
    load_bias<FULL>(p, c, bias);
    epi8<T, ACT, FULL>(p, v, r, c, n, rv, bias);
}
template <typename T, int ACT> __global__ __launch_bounds__(256) void linear_join_kernel(LinP p) { linear_join<T, ACT, true>(p, blockIdx.x); }

// ---- dz = dy act'(z), and the column sums of the unrounded dz: a block takes 256 V columns by RPB rows
struct DzP {
    const void *dy, *pre;
    long long ldy, ldpre;
    void* dz;       // [M][ldz], columns N .. ldz - 1 zero; NULL: only the sums
    float* part;    // [row blocks][N], or NULL
    int M, N, ldz, rows;
};
template <typename T, int V, int ACT> __device__ __forceinline__ void linear_dz(const DzP& p, int bx, int by, float* sm) {  // sm: 4 rows of 64 V + 1
    const int c = (bx * 64 + (threadIdx.x & 63)) * V, ty = threadIdx.x >> 6;
    const int row0 = by * p.rows, row1 = min(p.M, row0 + p.rows), width = p.dz ? p.ldz : p.N;
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
    for (int j = 0; j < V; j++) sm[ty * (64 * V + 1) + (threadIdx.x & 63) * V + j] = s[j];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * V; i += 256) {
        const int col = bx * 64 * V + i;
        constexpr int W = 64 * V + 1;
        if (col < p.N) p.part[(size_t)by * p.N + col] = (sm[i] + sm[W + i]) + (sm[2 * W + i] + sm[3 * W + i]);
    }
}
template <typename T, int V, int ACT> __global__ __launch_bounds__(256) void linear_dz_kernel(DzP p) {
    __shared__ float sm[4 * (64 * V + 1)];
    linear_dz<T, V, ACT>(p, blockIdx.x, blockIdx.y, sm);
}
__device__ __forceinline__ void linear_db(const float* part, float* db, int chunks, int N, int blk) {
    // 16 lanes x 16 columns: 16 strides of the chunks, joined in LDS in fp64
    __shared__ double sm[16][17];
    const int cx = threadIdx.x & 15, y = threadIdx.x >> 4, c = blk * 16 + cx;
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

// ---- the products of the backward in one launch: the blocks of dW, those of dx and, without an activation, those of the column sums of dy.
// Two 128 x 128 blocks per CU; one launch fills the chip where dW (few tiles, long k) or dx alone would not, and the tails overlap.
struct BwdP {
    LinP w, x;
    int wr, wc, xr, xc;           // tiles
    int n0, n1;                   // blocks of the first and of the first two segments (multiples of 8, so that block index modulo 8 stays the XCD)
    int w_first;                  // the segment with the longer blocks comes first
    DzP s;
    int sx;                       // column blocks of the sums
};
template <typename T, bool ALIGNED, int SV> __global__ __launch_bounds__(256, 2) void linear_bwd_kernel(BwdP p) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int id = blockIdx.x;
    if (id >= p.n1) {
        if constexpr (SV > 0) linear_dz<T, SV, ACT_NONE>(p.s, (id - p.n1) % p.sx, (id - p.n1) / p.sx, reinterpret_cast<float*>(smem));
        return;
    }
    const bool first = id < p.n0;
    const int at = first ? id : id - p.n0;
    if (first == (p.w_first != 0)) {
        if (at < p.wr * p.wc * p.w.splits) linear_tile<T, true, true, 128, 128, 2, 2, 2, ALIGNED, false>(p.w, p.wr, p.wc, at, smem);
    } else {
        if (at < p.xr * p.xc * p.x.splits) linear_tile<T, false, true, 128, 128, 2, 2, 2, ALIGNED, false>(p.x, p.xr, p.xc, at, smem);
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
template <typename T, int BR, int BC, int WR, int WC, int NS, int MINW, bool ALIGNED> int fwd_launch(const LinP& p, hipStream_t st) {
    constexpr size_t lds = lds_of<BR, BC, WR * WC, WC, ALIGNED ? NS : 1>();
    auto kern = linear_kernel<T, BR, BC, WR, WC, NS, MINW, ALIGNED>;
    if constexpr (lds > 64 * 1024) {
        static std::atomic<bool> set[64];
        const int rc = raise_lds(kern, lds, set);
        if (rc != DIG_OK) return rc;
    }
    const int rt = up(p.R, BR), ct = up(p.C, BC);
    hipLaunchKernelGGL(kern, dim3((unsigned)(rt * ct * p.splits)), dim3(WR * WC * 64), lds, st, p, rt, ct);
    if (p.splits > 1) {
        const dim3 grid((unsigned)(((long long)p.R * up(p.C, 8) + 255) / 256));
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

#ifndef FORCE_TILE
#define FORCE_TILE 0
#endif
enum { TILE_64 = 1, TILE_128 = 2, TILE_192 = 3, TILE_256 = 4 };
// tile and k slices of the forward
int fwd_plan(int M, int N, int K, int dtype, int& splits) {
    splits = 1;
    if (FORCE_TILE) return FORCE_TILE;
    return TILE_128;
}

// byte offsets inside a tile are 31 bits: up to 256 rows of a k-adjacent operand, the tile's k rows of the others
bool offsets_ok(long long ld, bool k_adjacent, int esize) { return ld * (k_adjacent ? 256 : KB / esize) * esize < (1ll << 31); }

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
    const bool aligned = a->K % E == 0 && a->ldx % E == 0 && a->ldw % E == 0 && al16(a->x) && al16(a->w) && offsets_ok(a->ldx, true, (int)sizeof(T)) &&
                         offsets_ok(a->ldw, true, (int)sizeof(T));
    int splits;
    const int tile = fwd_plan(a->M, a->N, a->K, a->dtype, splits);
    set_split(p, splits, KB / (int)sizeof(T));
    if (!aligned) return fwd_launch<T, 128, 128, 2, 2, 2, 2, false>(p, st);
    switch (tile) {
        case TILE_64: return fwd_launch<T, 64, 64, 2, 2, 4, 2, true>(p, st);
        case TILE_192: return fwd_launch<T, 192, 128, 2, 2, 2, 2, true>(p, st);
        case TILE_256: return fwd_launch<T, 256, 256, 2, 4, 2, 2, true>(p, st);
        default: return fwd_launch<T, 128, 128, 2, 2, 2, 2, true>(p, st);
    }
}

// ---- backward
// k slices of dx (nkx k tiles) and dW (nkw): least estimated time of one launch over 512 block slots, in k steps of a block.  A block costs its k tiles
// and OVER more (fill and epilogue); what is split is written and read again as fp32.
void bwd_plan(int M, int N, int K, int dtype, bool dx, int& sx, int& sw) {
    const int bk = KB / (dtype == DIG_BF16 ? 2 : 4), nkx = up(N, bk), nkw = up(M, bk);
    const double tx = dx ? (double)up(M, TILE) * up(K, TILE) : 0.0, tw = (double)up(N, TILE) * up(K, TILE), OVER = 4.0;
    const double join = dtype == DIG_BF16 ? 1.0 / (0.75 * 4.0e6) : 1.0 / (3.5 * 4.0e6);  // k steps per byte written and read: a step takes 0.75 (fp32: 3.5) us, a byte 0.25 ps
    double best = 1e30;
    sx = sw = 1;
    for (int a = 1; a <= 4 && (a == 1 || (dx && nkx >= 4 * a)); a++)
        for (int b = 1; b <= 64 && (b == 1 || nkw >= 4 * b); b++) {
            const double bx = up(nkx, a) + OVER, bw = up(nkw, b) + OVER, work = tx * a * bx + tw * b * bw, most = (dx && bx > bw) ? bx : bw;
            double t = work / 512.0 + 0.5 * most;
            if (t < most) t = most;
            if (a > 1) t += join * 4.0 * a * M * K * 2;
            if (b > 1) t += join * 4.0 * b * N * K * 2;
            if (t < best - 1e-9) {
                best = t;
                sx = a;
                sw = b;
            }
        }
    sx = up(nkx, up(nkx, sx));
    sw = up(nkw, up(nkw, sw));
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

template <typename T, int ACT> void dz_launch(const DzP& d, bool vec, dim3 grid, hipStream_t st) {
    if (vec) hipLaunchKernelGGL((linear_dz_kernel<T, 8, ACT>), grid, dim3(256), 0, st, d);
    else hipLaunchKernelGGL((linear_dz_kernel<T, 1, ACT>), grid, dim3(256), 0, st, d);
}

// floats of partial products of dx and dW
long long bwd_part(int M, int N, int K, int dtype, long long& dx_floats) {
    int sx, sw;
    bwd_plan(M, N, K, dtype, true, sx, sw);
    dx_floats = sx > 1 ? (long long)sx * M * K : 0;
    long long most = dx_floats + (sw > 1 ? (long long)sw * N * K : 0);
    bwd_plan(M, N, K, dtype, false, sx, sw);  // the same workspace serves a call without dx
    const long long alone = sw > 1 ? (long long)sw * N * K : 0;
    if (alone > most) most = alone;
    dx_floats = (dx_floats + 3) / 4 * 4;
    return (most + 7) / 4 * 4;
}

template <typename T> int bwd(const dig_linear_act_bwd_args* a, hipStream_t st) {
    const int E = 16 / (int)sizeof(T), es = (int)sizeof(T), M = a->M, N = a->N, K = a->K, ldz = up(N, 8) * 8;
    const int chunks = dz_chunks(M);
    long long xf;
    const long long pf = bwd_part(M, N, K, a->dtype, xf);
    float* sums = a->ws + pf;  // column sums of row blocks
    const DzP d{a->dy, a->pre, a->ldy, a->ldpre, a->dz, a->db ? sums : nullptr, M, N, ldz, dz_rows(M)};
    const bool dvec = N % 8 == 0 && a->ldy % 8 == 0 && al16(a->dy) && (a->act == ACT_NONE || (a->ldpre % 8 == 0 && al16(a->pre))) && (!a->dz || al16(a->dz));
    const int width = a->dz ? ldz : N, dcols = dvec ? up(width, 512) : up(width, 64);
    if (a->dz) {
        const dim3 grid((unsigned)dcols, (unsigned)chunks);
        switch (a->act) {
            case ACT_RELU: dz_launch<T, ACT_RELU>(d, dvec, grid, st); break;
            case ACT_GELU: dz_launch<T, ACT_GELU>(d, dvec, grid, st); break;
            case ACT_SILU: dz_launch<T, ACT_SILU>(d, dvec, grid, st); break;
            default: dz_launch<T, ACT_NONE>(d, dvec, grid, st); break;
        }
    }
    const void* dz = a->dz ? a->dz : a->dy;
    const long long lz = a->dz ? ldz : a->ldy;
    const bool aligned = lz % E == 0 && al16(dz) && (a->dz || N % E == 0) && K % E == 0 && a->ldx % E == 0 && al16(a->x) && offsets_ok(lz, true, es) && offsets_ok(a->ldx, false, es) &&
                         (!a->dx || (a->ldw % E == 0 && al16(a->w) && offsets_ok(a->ldw, false, es)));
    BwdP p{};
    int sx, sw;
    bwd_plan(M, N, K, a->dtype, a->dx != nullptr, sx, sw);
    p.w.p = p.x.p = dz;  // dW[n][k] = sum_m dz[m][n] x[m][k],  dx[m][k] = sum_n dz[m][n] W[n][k]
    p.w.ldp = p.x.ldp = lz;
    p.w.q = a->x;
    p.w.ldq = a->ldx;
    p.x.q = a->w;
    p.x.ldq = a->ldw;
    p.w.R = N;
    p.w.rpad = a->dz ? ldz : N;
    p.x.R = M;
    p.w.C = p.w.cpad = p.x.C = p.x.cpad = K;
    p.w.K = M;
    p.x.K = N;
    p.w.out = a->dw;
    p.x.out = a->dx;
    p.w.ldo = p.x.ldo = K;
    p.w.out_f32 = a->dw_f32;
    p.w.vec = K % 8 == 0 && al16(a->dw);
    p.x.vec = K % 8 == 0 && al16(a->dx);
    p.x.part = a->ws;
    p.w.part = a->ws + (a->dx ? xf : 0);
    set_split(p.w, sw, KB / es);
    set_split(p.x, sx, KB / es);
    p.wr = up(N, TILE);
    p.wc = p.xc = up(K, TILE);
    p.xr = a->dx ? up(M, TILE) : 0;
    p.w_first = !a->dx || p.w.kper >= p.x.kper;
    const int nw = up(p.wr * p.wc * p.w.splits, 8) * 8, nx = up(p.xr * p.xc * p.x.splits, 8) * 8;
    p.n0 = p.w_first ? nw : nx;
    p.n1 = nw + nx;
    const bool sum_here = a->db && !a->dz;
    p.s = d;
    p.sx = dcols;
    const dim3 grid((unsigned)(p.n1 + (sum_here ? dcols * chunks : 0)));
    constexpr size_t lds = lds_of<TILE, TILE, 4, 2, 2>();
    static_assert(lds <= 64 * 1024, "no attribute needed");
    if (aligned) {
        if (sum_here && dvec) hipLaunchKernelGGL((linear_bwd_kernel<T, true, 8>), grid, dim3(256), lds, st, p);
        else hipLaunchKernelGGL((linear_bwd_kernel<T, true, 1>), grid, dim3(256), lds, st, p);
    } else {
        if (sum_here && dvec) hipLaunchKernelGGL((linear_bwd_kernel<T, false, 8>), grid, dim3(256), lds, st, p);
        else hipLaunchKernelGGL((linear_bwd_kernel<T, false, 1>), grid, dim3(256), lds, st, p);
    }
    auto join_blocks = [](const LinP& q) { return q.splits > 1 ? (int)(((long long)q.R * up(q.C, 8) + 255) / 256) : 0; };
    const int jw = join_blocks(p.w), jx = a->dx ? join_blocks(p.x) : 0, jd = a->db ? up(N, 16) : 0;
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
extern "C" int dig_linear_act_bwd_ws(int M, int N, int K, int dtype) {
    if (!shape_ok(M, N, K) || !shape_ok(N, K, 1)) return DIG_EINVAL;
    long long xf;
    const long long n = bwd_part(M, N, K, dtype, xf) + (long long)dz_chunks(M) * N;
    return n < (1ll << 31) ? (int)n : DIG_EINVAL;
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
