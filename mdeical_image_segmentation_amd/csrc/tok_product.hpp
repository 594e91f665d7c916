// The kernel of the token products, any shape / stride / alignment: C[m][n] = sum_k A(m, k) B(n, k) (tok_gemm.hpp), included by one .hip per (type, tile).
//
// A block of 4 waves (2 x 2) owns a 32 FM x 32 FN piece of C, a wave FM x FN MFMA tiles of 16 x 16: 128 x 128 (two blocks per CU) where that fills the chip, 64 x 64 (four) for smaller
// products - gated 64 rows x 64 columns of gate and of up.
//
// A step is 128 bytes of k per row (64 bf16 / 32 f32), in two halves.  The pipeline of a wave, all of it plain code whose waits the compiler counts:
//      half 0   MFMAs of half 0 | fragments of half 1 <- LDS | step s + 1: registers -> other LDS buffer | step s + 2 or s + 3: global -> registers
//      barrier
//      half 1   MFMAs of half 1 | fragments of half 0 of step s + 1 <- other LDS buffer
// One barrier a step: a buffer is overwritten a step after its last reads, which were waited for in front of the barrier between.  The steps are flat over a block's tiles (the grid is what
// the chip holds at once), so the next tile's first steps are on their way while a finished tile is stored.
//
// B(n) feeds the MFMA's row side, A(m) its column side: a lane then holds runs of 8 consecutive n of one m, and bias, residual and stores are 16 bytes wide.
//   LDS image, k contiguous:   [row][128 B], 16-byte chunks at position c ^ key(row): a fragment read touches each bank once
//   LDS image, own index cont.: [k][TILE elements]; bf16 fragments by the transposing read (16 lanes: 4 k x 4 runs of 4), f32 ones by plain 16-byte reads, which give one k of four
//                              MFMA tiles (tile v then holds the indices 4 r + v)
// Bound, f32: the MFMAs (16 x 16 x 4, 32 cycles): 8192 x 1024 x 4096 510 us, 135 of the 154 TFLOP/s that a large f32 product of the library reaches.  bf16: two blocks' LDS traffic (as many bytes
// per MFMA and half as many again as the 256 x 256 tiles'): 2048^3 27 us, 0.63 PFLOP/s, where those tiles leave three quarters of the chip idle (45 us).  Operands at any address go by
// element-aligned loads with a mask per chunk: 2047 x 2049 x 2051 dz W 81 us against 50 with aligned copies.
// Sums are f32 (MFMA accumulators); k order inside a step is the same for both operands, which is all the sum needs.
#pragma once
#include "tok_epilogue.hpp"
#include "tok_product_plan.hpp"

namespace {
typedef __attribute__((address_space(3))) s16x4 tp_lds_s16x4;
constexpr int TP_OOB = (int)0xFFFFFF00u;          // past every buffer below: reads as zero

// swizzle keys.  Rows of a fragment: A side 16 f + li, B side 32 (f >> 1) + 8 (li >> 2) + 4 (f & 1) + (li & 3)
template <bool B> __device__ __forceinline__ int tp_key(int row) {
    return B ? (((row >> 1) & 1) | (((row >> 3) & 3) << 1)) : ((row >> 1) & 7);
}
// 32-byte position of a [k][i] bf16 row of TILE elements.  A side: a group of 16 lanes reads 32 bytes of 4 rows; B side: 8 of every 16 bytes of a 64-byte run of 4 rows.  (64 elements: two
// rows share the 256 bytes of the banks.)
template <bool B, int TILE> __device__ __forceinline__ int tp_pos32(int c32, int k) {
    if constexpr (TILE == 64) return B ? (c32 ^ (k & 2)) : (c32 ^ (((k >> 1) & 1) | (((k >> 3) & 1) << 1)));
    else return B ? (c32 ^ ((k & 3) << 1)) : (c32 ^ ((k & 3) | (((k >> 3) & 1) << 2)));
}
// one 16-byte chunk of which n elements exist, at any element address
template <typename T> __device__ __forceinline__ u32x4 tp_chunk(const T* p, long long n) {
    constexpr int EPC = Tr<T>::EPC;
    if (n >= EPC) return tok_ld16<T>(p);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n > 0) {
        float f[EPC];
#pragma unroll
        for (int i = 0; i < EPC; ++i) f[i] = i < n ? ld_elem<T>(p + i) : 0.f;
        v = pack_chunk<T>(f);
    }
    return v;
}

// one operand's step: origin of the tile at its first k, k and rows (own indices) present from there on (wave-uniform)
struct TpStep {
    const char* base;
    const char* base2;      // gated B: the up rows
    int left, rows;         // (rows: at most the tile's)
};

// Staging of one operand: F chunks of 16 bytes per thread.  k contiguous: chunk c = t & 7 of the rows (t >> 3) + 32 j; own index contiguous: chunk t % CPR of the k rows t / CPR + j KR.
template <typename T, bool MN, bool B, int EPI, bool AL, int F, int SETS> struct TpStage {
    static constexpr int ES = sizeof(T), EPC = Tr<T>::EPC, TILE = 32 * F, CPR = TILE / EPC, KR = 256 / CPR;
    static constexpr bool PAIR = B && EPI == TG_GATED;
    int c, r;               // chunk, first row / k row
    unsigned voff;          // byte offset of chunk 0 (AL)
    long long ld;
    u32x4 v[SETS][F];
    __device__ __forceinline__ TpStage(long long ld_) : ld(ld_) {
        const int t = threadIdx.x;
        c = MN ? t % CPR : t & 7;
        r = MN ? t / CPR : t >> 3;
        voff = (unsigned)(r * ld * ES) + c * 16;
    }
    // chunk j of the step; one that does not exist reads as zeros
    __device__ __forceinline__ void load(const TpStep& s, int set, int j) {
        if constexpr (AL) {
            // (chunks are whole here: a lane is in or out)
            const __amdgpu_buffer_rsrc_t q = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(PAIR && (j & 1) ? s.base2 : s.base), 0, 0x7fffffff, 0x00020000);
            const bool ok = MN ? (r + j * KR < s.left && c * EPC < s.rows) : (c * EPC < s.left && r + rowstep(j) < s.rows);
            v[set][j] = __builtin_amdgcn_raw_buffer_load_b128(q, ok ? (int)voff : TP_OOB, (int)(rowstep(j) * ld * ES), 0);
        } else {
            const T* p = reinterpret_cast<const T*>(PAIR && (j & 1) ? s.base2 : s.base) + (long long)(r + rowstep(j)) * ld + c * EPC;
            if constexpr (MN) v[set][j] = tp_chunk<T>(p, r + j * KR < s.left ? s.rows - c * EPC : 0);
            else v[set][j] = tp_chunk<T>(p, r + rowstep(j) < s.rows ? s.left - c * EPC : 0);
        }
    }
    static constexpr int TILE_K = Tr<T>::CK;
    // rows (k rows) that chunk j lies behind chunk 0; gated B: rows 64 b + q of the tile are column 32 b + (q & 31), of gate for q < 32, else of up
    static constexpr int rowstep(int j) { return MN ? j * KR : (PAIR ? (j >> 1) * 32 : j * 32); }
    __device__ __forceinline__ void put(char* lds, int set, int j) const {
        int off;
        if constexpr (!MN) {
            off = (r + 32 * j) * 128 + ((c ^ tp_key<B>(r)) << 4);          // (key(r + 32 j) = key(r))
        } else if constexpr (ES == 2) {
            const int k = r + j * KR;
            off = k * (TILE * 2) + (tp_pos32<B, TILE>(c >> 1, k) << 5) + ((c & 1) << 4);
        } else {
            off = (r + j * KR) * (TILE * 4) + c * 16;
        }
        lds_write_b128(lds, off, v[set][j]);
    }
};

// fragment f of a wave's 16 F rows (own indices) for half kk of a step; f32 with its own index contiguous: 16-byte reads give four fragments at once (asked for with f = 0)
template <typename T, bool MN, bool B, int F> __device__ __forceinline__ void tp_frag(u32x4 (&v)[F], const char* lds, int w, int kk, int f) {
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    constexpr int TILE = 32 * F;
    if constexpr (!MN) {
        const int row = w * 16 * F + (B ? 32 * (f >> 1) + 8 * (li >> 2) + 4 * (f & 1) + (li & 3) : 16 * f + li);
        v[f] = lds_read_b128(lds, row * 128 + (((kk * 4 + lg) ^ tp_key<B>(row)) << 4));
    } else if constexpr (sizeof(T) == 2) {
        const int i = w * 16 * F + (B ? 32 * (f >> 1) + 8 * (li & 3) + 4 * (f & 1) : 16 * f + 4 * (li & 3));
        s16x4 h[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k = kk * 32 + 8 * lg + 4 * s + (li >> 2);
            const uint32_t at = (uint32_t)(uintptr_t)lds + k * (TILE * 2) + (tp_pos32<B, TILE>(i >> 4, k) << 5) + ((i & 15) << 1);
            h[s] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tp_lds_s16x4*>(at));
        }
        const u32x2 lo = __builtin_bit_cast(u32x2, h[0]), hi = __builtin_bit_cast(u32x2, h[1]);
        v[f] = u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
        // 16 F own indices per wave: lane li holds the F indices F li ... of one k, tile q the q-th of them
        if (f != 0) return;
        float t[4][F];
#pragma unroll
        for (int s = 0; s < 4; ++s) __builtin_memcpy(t[s], __builtin_assume_aligned(lds + (kk * 16 + 4 * lg + s) * (TILE * 4) + (w * 16 * F + F * li) * 4, 4 * F), 4 * F);
#pragma unroll
        for (int q = 0; q < F; ++q) v[q] = u32x4{__float_as_uint(t[0][q]), __float_as_uint(t[1][q]), __float_as_uint(t[2][q]), __float_as_uint(t[3][q])};
    }
}

// B side index of value j (0..7) of run h of a lane: base(h) + j, held by tile f, accumulator q
template <typename T, bool BMN, int FN> struct TpRun {
    static constexpr bool R4 = BMN && sizeof(T) == 4;
    static __device__ __forceinline__ int base(int h, int lg) { return R4 ? 4 * FN * lg + 8 * h : 32 * h + 8 * lg; }
    static constexpr int f(int h, int j) { return R4 ? (8 * h + j) % FN : 2 * h + (j >> 2); }
    static constexpr int q(int h, int j) { return R4 ? (8 * h + j) / FN : (j & 3); }
};
}   // namespace

constexpr int tp_blocks(int fm, int fn) { return fm == 4 ? 2 : (fn == 4 ? 3 : 4); }          // per CU

template <typename T, bool AMN, bool BMN, int EPI, bool AL, int FM, int FN>
__global__ __launch_bounds__(256, tp_blocks(FM, FN)) void tok_product_kernel(const TgArgs a, const TpPlan pl) {
    constexpr int CK = Tr<T>::CK, ES = sizeof(T), TM = 32 * FM, TN = 32 * FN, BN = EPI == TG_GATED ? TN / 2 : TN, OPA = TM * 128, STAGE = OPA + TN * 128;
    static_assert(FM <= FN, "");
    extern __shared__ __attribute__((aligned(1024))) char smem[];          // 2 x [A | B]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int li = lane & 15, lg = lane >> 4;
    const int first = xcd_remap(blockIdx.x, gridDim.x);
    if (first >= pl.items) return;                            // block-uniform
    const int tiles = pl.tm * pl.tn, all_steps = a.ranges * pl.spr;

    // items: batch-major, then k part, then tile; tiles in bands of 4 tile rows, column by column inside a band (the neighbours that run on an XCD share row and column panels in its L2)
    auto tile_of = [&](int it) __attribute__((always_inline)) {
        TpItem w;
        const int bs = it / tiles, t = it - bs * tiles;
        w.bt = bs / pl.splits;
        w.sp = bs - w.bt * pl.splits;
        const int band = t / (4 * pl.tn), in = t - band * 4 * pl.tn;
        const int h = pl.tm - band * 4 < 4 ? pl.tm - band * 4 : 4;
        const int c = in / h;
        w.m0 = (long long)(band * 4 + in - c * h) * TM;
        w.n0 = (long long)c * BN;
        return w;
    };
    // (an item has an even number of steps, the last of an odd number reads nothing but zeros: the loop below is two steps long)
    auto steps_of = [&](int sp) __attribute__((always_inline)) { return all_steps - sp * pl.sps < pl.sps ? all_steps - sp * pl.sps : pl.sps; };

    // ---- load cursor: the step that goes into the staging registers next ----
    // Steps that wait in registers: two (2048^3 bf16 dz W 31 -> 27 us, 64 x 64 tiles 5 to 15 %, f32 2 to 4 %) where they fit - operands at any address, bf16 dz^T x in 128 x 128 tiles and gated
    // 64 x (64 + 64) spill with them (8192 x 1024 x 4096: 88 -> 111 us, gated 175 -> 312)
    constexpr int SETS = AL && !(EPI == TG_GATED && FM == 2) && !(AMN && ES == 2 && FM == 4) ? 2 : 1;
    TpStage<T, AMN, false, EPI, AL, FM, SETS> ga(a.a.ld);
    TpStage<T, BMN, true, EPI, AL, FN, SETS> gb(a.b.ld);
    TpStep na, nb;
    int lit = first, lrem = 0, lpad = 0;
    const long long step_a = AMN ? CK * ES * a.a.ld : CK * ES, step_b = BMN ? CK * ES * a.b.ld : CK * ES;
    auto place = [&](long long m0, long long n0, int bt, int at) __attribute__((always_inline)) {
        const int range = at >= pl.spr ? 1 : 0, ks = at - range * pl.spr;
        // (p + s (p2 - p), not s ? p2 : p: hipcc turns that into an indexed load from a scratch copy of the arguments)
        const long long da = (const char*)a.a.p2 - (const char*)a.a.p, db = (const char*)a.b.p2 - (const char*)a.b.p;
        na.base = (const char*)a.a.p + (EPI == TG_GATED ? 0 : bt | range) * da + (AMN ? m0 : m0 * a.a.ld) * ES + ks * step_a;
        nb.base = (const char*)a.b.p + (EPI == TG_GATED ? 0 : bt | range) * db + (BMN ? n0 : n0 * a.b.ld) * ES + ks * step_b;
        nb.base2 = nb.base + db;
        na.left = nb.left = (int)(a.K - (long long)ks * CK);
        na.rows = a.M - m0 < TM ? (int)(a.M - m0) : TM;
        nb.rows = a.N - n0 < BN ? (int)(a.N - n0) : BN;
    };
    // the first step of item lit, or (second) of its second range; behind the last item: rows 0, everything reads as zeros (by a select - stores of the fields in two branches become
    // one store through a pointer to scratch, and its reload every step waits for
    // the prefetch: 32768 x 1024 x 4096 in 128 x 128 tiles 383 us instead of 344)
    auto load_tile = [&](bool second) __attribute__((always_inline)) {
        const bool live = lit < pl.items;
        const TpItem w = tile_of(live ? lit : first);
        const int n = steps_of(w.sp);
        lrem = second ? lrem : n + (n & 1);
        lpad = n & 1;
        place(w.m0, w.n0, w.bt, second ? pl.spr : w.sp * pl.sps);
        na.rows = live ? na.rows : 0;
        nb.rows = live ? nb.rows : 0;
    };
    auto advance = [&]() __attribute__((always_inline)) {
        na.base += step_a;
        nb.base += step_b;
        nb.base2 += step_b;
        na.left -= CK;
        nb.left -= CK;
        --lrem;
        if (lrem == lpad) na.left = nb.left = lrem == 0 ? na.left : 0;
        if (lrem == 0 || (na.left <= 0 && lrem != lpad)) {
            lit += lrem == 0 ? (int)gridDim.x : 0;
            load_tile(lrem != 0);
            __builtin_amdgcn_s_waitcnt(0xc07f);               // (lgkmcnt(0): a scalar load in flight here would turn the loop's waits for LDS reads into waits for all of them)
        }
    };

    f32x4 acc[FN][FM];
#pragma unroll
    for (int f = 0; f < FN; ++f)
#pragma unroll
        for (int p = 0; p < FM; ++p) acc[f][p] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto barrier = [&]() __attribute__((always_inline)) {     // this wave's LDS traffic is done, then everyone's is; loads from global memory stay in flight
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    load_tile(false);
    // chunk f of both operands (FM <= FN)
    auto load = [&](int set, int f) __attribute__((always_inline)) {
        if (f < FM) ga.load(na, set, f);
        gb.load(nb, set, f);
    };
    auto put = [&](char* st, int set, int f) __attribute__((always_inline)) {
        if (f < FM) ga.put(st, set, f);
        gb.put(st + OPA, set, f);
    };
    u32x4 a0[FM], b0[FN], a1[FM], b1[FN];
    // fragments 2 f, 2 f + 1 of half kk
    auto frags = [&](u32x4 (&av)[FM], u32x4 (&bv)[FN], const char* st, int kk, int f) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 2 * f; g < 2 * f + 2; ++g) {
            if (g < FM) tp_frag<T, AMN, false, FM>(av, st, wm, kk, g);
            if (g < FN) tp_frag<T, BMN, true, FN>(bv, st + OPA, wn, kk, g);
        }
    };
    // steps 0 .. SETS on their way, step 0 into LDS
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
#pragma unroll
        for (int f = 0; f < FN; ++f) load(s, f);
        advance();
    }
#pragma unroll
    for (int f = 0; f < FN; ++f) {
        put(smem, 0, f);
        load(0, f);
    }
    advance();
    barrier();
#pragma unroll
    for (int f = 0; f < FN; ++f) frags(a0, b0, smem, 0, f);

    int cit = first;
    TpItem ct = tile_of(cit);
    int crem = steps_of(ct.sp);
    while (true) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {                         // steps of even and odd number: buffers and register sets by name
            char* const cur = smem + p * STAGE;
            char* const nxt = smem + (p ^ 1) * STAGE;
            const int set = (p ^ 1) & (SETS - 1);
            // (sched_barrier: the scheduler interleaves inside a row of MFMAs but does not pull a whole step's loads together, which would not fit the registers)
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                frags(a1, b1, cur, 1, f);
                put(nxt, set, f);
                load(set, f);
#pragma unroll
                for (int q = 0; q < FM; ++q) mma_b128<T>(acc[f][q], b0[f], a0[q]);
                __builtin_amdgcn_sched_barrier(0);
            }
            advance();
            barrier();
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                frags(a0, b0, nxt, 0, f);
#pragma unroll
                for (int q = 0; q < FM; ++q) mma_b128<T>(acc[f][q], b1[f], a1[q]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if ((crem -= 2) > 0) continue;

        // ---- the tile is complete ----
        using Run = TpRun<T, BMN, FN>;
        if constexpr (EPI == TG_GATED) {
            // MFMA tiles 0, 1 hold 8 gate columns of a lane, 2, 3 the same columns of up
            static_assert(!Run::R4 && FN == 4, "gated: k-contiguous weights, 64 B rows per wave");
            const TgGatedRow<T> row(a, ct.n0 + wn * 32 + 8 * lg);
            if (row.nv > 0) {
#pragma unroll
                for (int p = 0; p < FM; ++p) {
                    const long long m = ct.m0 + wm * 16 * FM + 16 * p + li;
                    float g[8], u[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        g[j] = acc[j >> 2][p][j & 3];
                        u[j] = acc[2 + (j >> 2)][p][j & 3];
                    }
                    if (m < a.M) row(m, g, u);
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < FN / 2; ++h) {
                const long long n = ct.n0 + wn * 16 * FN + Run::base(h, lg);
                const TgLinearRow<T> row(a, tg_out(a, ct.bt), n, EPI == TG_LINEAR);
                float* const sl = pl.slab + (long long)(ct.bt * pl.splits + ct.sp) * a.M * a.N + n;
                if (row.nv > 0) {
#pragma unroll
                    for (int p = 0; p < FM; ++p) {
                        const long long m = ct.m0 + wm * 16 * FM + ((AMN && ES == 4) ? FM * li + p : 16 * p + li);
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = acc[Run::f(h, j)][p][Run::q(h, j)];
                        if (m < a.M) {
                            if constexpr (EPI == TG_LINEAR) row(m, v);
                            else if constexpr (EPI == TG_STORE) row.store(m, v);
                            else tok_stn<float>(sl + m * a.N, v, row.nv);
                        }
                    }
                }
            }
        }
        cit += gridDim.x;
        if (cit >= pl.items) return;
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
            for (int p = 0; p < FM; ++p) acc[f][p] = f32x4{0.f, 0.f, 0.f, 0.f};
        ct = tile_of(cit);
        crem = steps_of(ct.sp);
        __builtin_amdgcn_s_waitcnt(0xc07f);                   // (as above)
    }
}

namespace {
template <typename T, bool AMN, bool BMN, int EPI, bool AL, int F> int tp_go(const TgArgs& a, const TpPlan& pl, hipStream_t stream) {
    constexpr int FM = F, FN = EPI == TG_GATED ? 4 : F;
    constexpr size_t LDS = 2 * 32 * (FM + FN) * 128;          // at most 64 KiB
    constexpr int hold = 256 * tp_blocks(FM, FN);             // blocks that the chip holds at once
    hipLaunchKernelGGL((tok_product_kernel<T, AMN, BMN, EPI, AL, FM, FN>), dim3((unsigned)(pl.items < hold ? pl.items : hold)), dim3(256), LDS, stream, a, pl);
    MIS_LAUNCH_CHECK("token product");
    return MIS_OK;
}
template <typename T, int F, bool AL> int tp_pick(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream) {
    if (epi == TG_GATED) return tp_go<T, false, false, TG_GATED, AL, F>(a, pl, stream);
    if (epi == TG_LINEAR) return tp_go<T, false, false, TG_LINEAR, AL, F>(a, pl, stream);
    if (!b_mn) return tp_go<T, false, false, TG_SLAB, AL, F>(a, pl, stream);
    if (epi == TG_STORE) return a_mn ? tp_go<T, true, true, TG_STORE, AL, F>(a, pl, stream) : tp_go<T, false, true, TG_STORE, AL, F>(a, pl, stream);
    return a_mn ? tp_go<T, true, true, TG_SLAB, AL, F>(a, pl, stream) : tp_go<T, false, true, TG_SLAB, AL, F>(a, pl, stream);
}
}   // namespace
