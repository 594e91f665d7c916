// Large bf16 matrix products of the token operators: a persistent 256 x 256 ping-pong kernel, all three operand layouts (tok_gemm.hpp), 16-byte aligned operands.
//
// 8 waves, 2 (m) x 4 (n), a wave owns 128 x 64 of C as 8 x 4 MFMA tiles of 16 x 16 (128 accumulator registers).  A step is 64 k: two segments of 12 fragments (24 KiB of LDS reads per
// wave and step for 64 MFMAs) - the two waves of a SIMD are one barrier apart, so that one is always inside its 32 MFMAs (512 cycles) while the other fetches fragments:
//
//      slot        0            1            2            3               4
//      group 0     R0 B(s+1)    M0           R1 A(s+2)    M1 wait         R0' ...      R = fragment reads, M = 32 MFMAs, every slot ends with a barrier of all 8 waves
//      group 1     M1"          R0 B(s+1)    M0           R1 A(s+2) wait  M1 ...
//
// Both operands arrive by LDS-DMA, 64 KiB a step, four instructions of 1 KiB per wave in each of its R segments: the CU's load path takes about 25 cycles for one, and a wave that
// issues into the full path stalls (two of them inside an M segment made it 800 cycles long).  B is double-buffered and fetched one step ahead, A has three buffers and is fetched two
// steps ahead (all 160 KiB of LDS); a buffer's last readers passed the barrier in front of the slot that refills it, and slot 3 retires step s + 1 by a counted wait that leaves the
// four A(s+2) in flight.  The step sequence is flat over a block's tiles (grid = number of CUs), so a tile's first steps are in flight while the tile before is finished and stored.
// LDS images and swizzles are those of tok_gemm.hip with 256 rows: [row][128 B] for a k-contiguous operand, [k][512 B] for the other kind, read with the transposing ds_read_b64_tr_b16.
// The fragment reads and their wait are one asm statement: hipcc would put a vmcnt(0), i.e. a wait for the prefetch, in front of a plain LDS read while an LDS-DMA is in flight.
#include <stdlib.h>

#include "conv_pp_common.hpp"
#include "dispatch_cfg.hpp"
#include "tok_epilogue.hpp"

namespace {
constexpr int PG_OP = 32768;              // bytes of one operand's 64-k step
constexpr int PG_B0 = 3 * PG_OP;          // LDS: three A buffers, two B buffers
constexpr int PG_LDS = 5 * PG_OP;

struct PgPlan {
    int tm, tn;             // tiles of a product
    int splits;             // parts of the k steps (SLAB only, else 1)
    int spr;                // steps of one range: ceil(K / 64)
    int sps;                // steps of one split
    int items;              // batches * splits * tm * tn
    float* slab;            // SLAB: [batch][split][M][N] f32
};

// Fragments of one segment.  aA / aB: this lane's LDS address of fragment 0.
__device__ __forceinline__ void pg_read_kk(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB) {
    asm volatile(
        "ds_read_b128 %0, %13\n\tds_read_b128 %1, %13 offset:512\n\tds_read_b128 %2, %13 offset:4096\n\tds_read_b128 %3, %13 offset:4608\n\t"
        "ds_read_b128 %4, %12\n\tds_read_b128 %5, %12 offset:2048\n\tds_read_b128 %6, %12 offset:4096\n\tds_read_b128 %7, %12 offset:6144\n\t"
        "ds_read_b128 %8, %12 offset:8192\n\tds_read_b128 %9, %12 offset:10240\n\tds_read_b128 %10, %12 offset:12288\n\tds_read_b128 %11, %12 offset:14336\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(B[0]), "=&v"(B[1]), "=&v"(B[2]), "=&v"(B[3]), "=&v"(A[0]), "=&v"(A[1]), "=&v"(A[2]), "=&v"(A[3]), "=&v"(A[4]), "=&v"(A[5]), "=&v"(A[6]), "=&v"(A[7])
        : "v"(aA), "v"(aB)
        : "memory");
}
__device__ __forceinline__ u32x4 pg_join(const u32x2& lo, const u32x2& hi) { return u32x4{lo[0], lo[1], hi[0], hi[1]}; }
// B with its own index contiguous: fragment f at aB ^ (64 if f >= 2), + 8 bytes if f is odd; the second half of its k 4 rows (2048 B) further
__device__ __forceinline__ void pg_read_km(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB) {
    u32x2 b[8];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %17\n\tds_read_b64_tr_b16 %1, %17 offset:2048\n\tds_read_b64_tr_b16 %2, %17 offset:8\n\tds_read_b64_tr_b16 %3, %17 offset:2056\n\t"
        "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %18 offset:2048\n\tds_read_b64_tr_b16 %6, %18 offset:8\n\tds_read_b64_tr_b16 %7, %18 offset:2056\n\t"
        "ds_read_b128 %8, %16\n\tds_read_b128 %9, %16 offset:2048\n\tds_read_b128 %10, %16 offset:4096\n\tds_read_b128 %11, %16 offset:6144\n\t"
        "ds_read_b128 %12, %16 offset:8192\n\tds_read_b128 %13, %16 offset:10240\n\tds_read_b128 %14, %16 offset:12288\n\tds_read_b128 %15, %16 offset:14336\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(b[4]), "=&v"(b[5]), "=&v"(b[6]), "=&v"(b[7]), "=&v"(A[0]), "=&v"(A[1]), "=&v"(A[2]), "=&v"(A[3]),
          "=&v"(A[4]), "=&v"(A[5]), "=&v"(A[6]), "=&v"(A[7])
        : "v"(aA), "v"(aB), "v"(aB ^ 64u)
        : "memory");
#pragma unroll
    for (int f = 0; f < 4; ++f) B[f] = pg_join(b[2 * f], b[2 * f + 1]);
}
// both of the other kind: A's fragment p at aA ^ (32 p)
__device__ __forceinline__ void pg_read_mm(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB) {
    u32x2 b[8], a[16];
    uint32_t t;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %26\n\tds_read_b64_tr_b16 %1, %26 offset:2048\n\tds_read_b64_tr_b16 %2, %26 offset:8\n\tds_read_b64_tr_b16 %3, %26 offset:2056\n\t"
        "ds_read_b64_tr_b16 %4, %27\n\tds_read_b64_tr_b16 %5, %27 offset:2048\n\tds_read_b64_tr_b16 %6, %27 offset:8\n\tds_read_b64_tr_b16 %7, %27 offset:2056\n\t"
        "ds_read_b64_tr_b16 %8, %25\n\tds_read_b64_tr_b16 %9, %25 offset:2048\n\t"
        "v_xor_b32 %24, 32, %25\n\tds_read_b64_tr_b16 %10, %24\n\tds_read_b64_tr_b16 %11, %24 offset:2048\n\t"
        "v_xor_b32 %24, 64, %25\n\tds_read_b64_tr_b16 %12, %24\n\tds_read_b64_tr_b16 %13, %24 offset:2048\n\t"
        "v_xor_b32 %24, 0x60, %25\n\tds_read_b64_tr_b16 %14, %24\n\tds_read_b64_tr_b16 %15, %24 offset:2048\n\t"
        "v_xor_b32 %24, 0x80, %25\n\tds_read_b64_tr_b16 %16, %24\n\tds_read_b64_tr_b16 %17, %24 offset:2048\n\t"
        "v_xor_b32 %24, 0xa0, %25\n\tds_read_b64_tr_b16 %18, %24\n\tds_read_b64_tr_b16 %19, %24 offset:2048\n\t"
        "v_xor_b32 %24, 0xc0, %25\n\tds_read_b64_tr_b16 %20, %24\n\tds_read_b64_tr_b16 %21, %24 offset:2048\n\t"
        "v_xor_b32 %24, 0xe0, %25\n\tds_read_b64_tr_b16 %22, %24\n\tds_read_b64_tr_b16 %23, %24 offset:2048\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(b[4]), "=&v"(b[5]), "=&v"(b[6]), "=&v"(b[7]), "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]),
          "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7]), "=&v"(a[8]), "=&v"(a[9]), "=&v"(a[10]), "=&v"(a[11]), "=&v"(a[12]), "=&v"(a[13]), "=&v"(a[14]), "=&v"(a[15]), "=&v"(t)
        : "v"(aA), "v"(aB), "v"(aB ^ 64u)
        : "memory");
#pragma unroll
    for (int f = 0; f < 4; ++f) B[f] = pg_join(b[2 * f], b[2 * f + 1]);
#pragma unroll
    for (int p = 0; p < 8; ++p) A[p] = pg_join(a[2 * p], a[2 * p + 1]);
}

// Where this lane's 16 bytes of an operand's DMA instructions lie, relative to the step's first element
struct PgLane {
    unsigned v0;            // byte offset in the wave's first instruction
    unsigned jstep;         // ... and between its four instructions: 64 rows (gated B: 32 columns) or 16 k further
    int row;                // k contiguous: row of the first instruction; else first column of the chunk
    int k;                  // k contiguous: first k of the chunk; else k row of the first instruction
};
// one operand's 64-k step (wave-uniform)
struct PgStep {
    const char* base;
    int left;               // k present, 64 or fewer
    int rows;               // tile rows (columns) present
    int whole;              // all of both
};

// The wave's four instructions of a step.  Valid lanes are inside the operand by construction; a lane that has to read zeros carries an offset past num_records.
template <bool MN, int RSTEP> __device__ __forceinline__ void pg_issue(const PgLane& l, const PgStep& s, char* dst, int wave) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(s.base), 0, 0x7fffffff, 0x00020000);
    if (s.whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) pp_dma16s(r, (int)l.v0, (int)(j * l.jstep), dst + (wave + 8 * j) * 1024);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool ok = MN ? (l.k + 16 * j < s.left && l.row < s.rows) : (l.k < s.left && l.row + RSTEP * j < s.rows);
            pp_dma16s(r, ok ? (int)l.v0 : PP_OOB, (int)(j * l.jstep), dst + (wave + 8 * j) * 1024);
        }
    }
}
}   // namespace

template <bool AMN, bool BMN, int EPI>
__global__ __launch_bounds__(512, 2) void tg_pp_kernel(const TgArgs a, const PgPlan pl) {
    using T = __bf16;
    constexpr int BN = EPI == TG_GATED ? 128 : 256;          // columns of C a tile covers
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int grp = wave >> 2, wm = wave >> 2, wn = wave & 3;
    const int li = lane & 15, lg = lane >> 4;

    const int first = xcd_remap(blockIdx.x, gridDim.x);
    if (first >= pl.items) return;                            // block-uniform
    const int tiles = pl.tm * pl.tn;
    const int nsteps_all = a.ranges * pl.spr;

    // ---- fragment addresses inside a stage ----
    uint32_t fA, fB;
    if constexpr (!AMN) fA = wm * 16384 + li * 128 + ((lg ^ (li >> 1)) << 4);
    else fA = (8 * lg + (li >> 2)) * 512 + ((wm * 8 + ((li >> 2) | ((lg & 1) << 2))) << 5) + 8 * (li & 3);
    if constexpr (!BMN) fB = PG_B0 + wn * 8192 + (8 * (li >> 2) + (li & 3)) * 128 + ((lg ^ (((li >> 1) & 1) | ((li >> 2) << 1))) << 4);
    else fB = PG_B0 + (8 * lg + (li >> 2)) * 512 + (((wn * 4 + ((li & 3) >> 1)) ^ ((li >> 2) << 1)) << 5) + 16 * (li & 1);

    // ---- DMA source offsets of this lane ----
    PgLane la, lb;
    constexpr int BROWS = EPI == TG_GATED ? 32 : 64;          // B rows (columns of C) an instruction index adds
    if constexpr (!AMN) {
        const int r = 8 * wave + (lane >> 3);                 // (+ 64 j)
        la.row = r;
        la.k = ((lane & 7) ^ ((r >> 1) & 7)) * 8;
        la.v0 = (unsigned)(r * a.a.ld + la.k) * 2;
        la.jstep = (unsigned)(128 * a.a.ld);
    } else {
        const int k = 2 * wave + (lane >> 5);                 // (+ 16 j)
        la.k = k;
        la.row = (((lane & 31) >> 1) ^ ((k & 3) | (((k >> 3) & 1) << 2))) * 16 + (lane & 1) * 8;
        la.v0 = (unsigned)(k * a.a.ld + la.row) * 2;
        la.jstep = (unsigned)(32 * a.a.ld);
    }
    if constexpr (!BMN) {
        const int r = 8 * wave + (lane >> 3);
        lb.row = EPI == TG_GATED ? (r & 31) : r;              // gated: rows 64 j + r of the tile hold column 32 j + (r & 31), of gate for r < 32 (waves 0..3), else of up
        lb.k = ((lane & 7) ^ (((r >> 1) & 1) | (((r >> 3) & 3) << 1))) * 8;
        lb.v0 = (unsigned)(lb.row * a.b.ld + lb.k) * 2;
        lb.jstep = (unsigned)(2 * BROWS * a.b.ld);
    } else {
        const int k = 2 * wave + (lane >> 5);
        lb.k = k;
        lb.row = (((lane & 31) >> 1) ^ ((k & 3) << 1)) * 16 + (lane & 1) * 8;
        lb.v0 = (unsigned)(k * a.b.ld + lb.row) * 2;
        lb.jstep = (unsigned)(32 * a.b.ld);
    }

    // items: batch-major, then k part, then tile; tiles in bands of 4 tile rows, column by column inside a band (32 neighbours of an XCD share 4 row panels and 8 column panels in its L2)
    auto tile_of = [&](int it, int& bt, int& sp, long long& m0, long long& n0) {
        const int t = it % tiles, bs = it / tiles;
        sp = bs % pl.splits;
        bt = bs / pl.splits;
        const int band = t / (4 * pl.tn), in = t - band * 4 * pl.tn;
        const int h = pl.tm - band * 4 < 4 ? pl.tm - band * 4 : 4;
        const int c = in / h;
        m0 = (long long)(band * 4 + in - c * h) * 256;
        n0 = (long long)c * BN;
    };
    auto steps_of = [&](int sp) {
        const int s0 = sp * pl.sps;
        return nsteps_all - s0 < pl.sps ? nsteps_all - s0 : pl.sps;
    };

    // ---- load cursor: `na` is the step whose A is issued next, `nb` the one whose B is (the step before, once the pipeline runs) ----
    int lit = first, lrange = 0, lrem = 0, krem = 0;          // item, range, steps of the item from the cursor's on, k of the range from the cursor's on
    PgStep na, nb, nb1;                                       // nb1: B of na's step
    bool va = true, vb = true;                                // whether na / nb is a step of this block
    const long long step_a = AMN ? 128 * a.a.ld : 128, step_b = BMN ? 128 * a.b.ld : 128;
    auto flags = [&]() __attribute__((always_inline)) {
        na.left = nb1.left = krem < 64 ? krem : 64;
        na.whole = na.left == 64 && na.rows == 256;
        nb1.whole = nb1.left == 64 && nb1.rows == BN;
    };
    // (tile, k part) of item lit at step `at` of its product -> na, nb1
    auto place = [&](long long m0, long long n0, int bt, int at) {
        lrange = at >= pl.spr ? 1 : 0;
        const int ks = at - lrange * pl.spr;
        // (p + s (p2 - p), not s ? p2 : p: hipcc turns that into an indexed load from a scratch copy of the arguments)
        const char* const pa = (const char*)a.a.p + (long long)(AMN ? bt : lrange) * ((const char*)a.a.p2 - (const char*)a.a.p);
        const char* const pb = (const char*)a.b.p + (long long)(EPI == TG_GATED ? (wave >> 2) : lrange) * ((const char*)a.b.p2 - (const char*)a.b.p);
        na.base = pa + (AMN ? m0 : m0 * a.a.ld) * 2 + ks * step_a;
        nb1.base = pb + (BMN ? n0 : n0 * a.b.ld) * 2 + ks * step_b;
        krem = (int)a.K - ks * 64;
        na.rows = a.M - m0 < 256 ? (int)(a.M - m0) : 256;
        nb1.rows = a.N - n0 < BN ? (int)(a.N - n0) : BN;
        flags();
    };
    auto load_tile = [&]() {
        int bt, sp;
        long long m0, n0;
        tile_of(lit, bt, sp, m0, n0);
        lrem = steps_of(sp);
        place(m0, n0, bt, sp * pl.sps);
    };
    auto advance = [&]() __attribute__((always_inline)) {     // A of the cursor's step is issued: its B is next, and A of the step behind it
        nb = nb1;
        vb = va;
        if (!va) return;
        na.base += step_a;
        nb1.base += step_b;
        krem -= 64;
        if (--lrem == 0) {
            lit += gridDim.x;
            va = lit < pl.items;
            if (va) load_tile();
        } else if (krem <= 0) {                               // the second range of the same tile
            int bt, sp;
            long long m0, n0;
            tile_of(lit, bt, sp, m0, n0);
            place(m0, n0, bt, pl.spr);
        } else {
            flags();
        }
    };
    load_tile();

    f32x4 acc[4][8];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int p = 0; p < 8; ++p) acc[f][p] = f32x4{0.f, 0.f, 0.f, 0.f};

    int sA = 0, sB = 0;                                       // buffers of the current step
    auto a_buf = [&](int ahead) { return smem + (sA + ahead >= 3 ? sA + ahead - 3 : sA + ahead) * PG_OP; };
    auto b_buf = [&](int ahead) { return smem + PG_B0 + ((sB + ahead) & 1) * PG_OP; };
    auto issue_a = [&](char* dst) __attribute__((always_inline)) { pg_issue<AMN, 64>(la, na, dst, wave); };
    auto issue_b = [&](char* dst) __attribute__((always_inline)) { pg_issue<BMN, BROWS>(lb, nb, dst, wave); };
    issue_a(smem);
    advance();
    issue_b(smem + PG_B0);
    if (va) issue_a(a_buf(1));                                // A of step 1
    advance();                                                // nb: B of step 1, na: A of step 2
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (grp == 1) __builtin_amdgcn_s_barrier();               // the stagger
    __builtin_amdgcn_sched_barrier(0);

    int cit = first, crem, bt, sp;
    long long m0, n0;
    tile_of(cit, bt, sp, m0, n0);
    crem = steps_of(sp);

    u32x4 fa[8], fb[4];
    auto read = [&](int kk) {
        // k-contiguous: the second half of the step is 64 bytes further in the row, i.e. chunk position ^ 4; else 32 k rows further
        const uint32_t xa = (uint32_t)(uintptr_t)smem + sA * PG_OP + (AMN ? fA + kk * 16384 : fA ^ (kk * 64));
        const uint32_t xb = (uint32_t)(uintptr_t)smem + sB * PG_OP + (BMN ? fB + kk * 16384 : fB ^ (kk * 64));
        if constexpr (!AMN && !BMN) pg_read_kk(fa, fb, xa, xb);
        else if constexpr (!AMN) pg_read_km(fa, fb, xa, xb);
        else pg_read_mm(fa, fb, xa, xb);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto mma = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int p = 0; p < 8; ++p) mma_b128<T>(acc[f][p], fb[f], fa[p]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto barrier = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    // step s + 1 is complete once at most the four A(s + 2) just issued are in flight
    auto retire = [&](bool inflight) __attribute__((always_inline)) {
        if (inflight) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };

#pragma unroll 1
    while (true) {
        // ---- segment 0 ----
        if (vb) issue_b(b_buf(1));
        else __builtin_amdgcn_s_sleep(1);                     // keep a distance between the barrier that published this step and its first read
        __builtin_amdgcn_sched_barrier(0);
        read(0);
        barrier();
        mma();
        barrier();
        // ---- segment 1 ----
        const bool inflight = va;
        if (va) issue_a(a_buf(2));
        __builtin_amdgcn_sched_barrier(0);
        read(1);
        advance();
        if (grp == 1) retire(inflight);
        barrier();
        mma();
        if (grp == 0) retire(inflight);
        barrier();
        sA = sA == 2 ? 0 : sA + 1;
        sB ^= 1;
        if (--crem == 0) {
            // ---- this wave's part of the tile is complete ----
            if constexpr (EPI == TG_GATED) {
                const TgGatedRow<T> row(a, n0 + wn * 32 + 8 * lg);
                if (row.nv > 0) {
#pragma unroll
                    for (int p = 0; p < 8; ++p) {
                        const long long m = m0 + wm * 128 + 16 * p + li;
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
                for (int h = 0; h < 2; ++h) {
                    const long long n = n0 + wn * 64 + 32 * h + 8 * lg;
                    if constexpr (EPI == TG_LINEAR) {
                        const TgLinearRow<T> row(a, a.y, n);
                        if (row.nv > 0) {
#pragma unroll
                            for (int p = 0; p < 8; ++p) {
                                const long long m = m0 + wm * 128 + 16 * p + li;
                                float v[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] = acc[2 * h + (j >> 2)][p][j & 3];
                                if (m < a.M) row(m, v);
                            }
                        }
                    } else {
                        const int nv = a.N - n >= 8 ? 8 : (int)(a.N - n);
                        if (nv > 0) {
                            T* const y = reinterpret_cast<T*>(bt == 0 ? a.y : a.y2) + n;
                            float* const sl = pl.slab + ((long long)(bt * pl.splits + sp) * a.M) * a.N + n;
#pragma unroll
                            for (int p = 0; p < 8; ++p) {
                                const long long m = m0 + wm * 128 + 16 * p + li;
                                float v[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] = acc[2 * h + (j >> 2)][p][j & 3];
                                if (m < a.M) {
                                    if constexpr (EPI == TG_STORE) tok_stn<T>(y + m * a.ldy, v, nv);
                                    else tok_stn<float>(sl + m * a.N, v, nv);
                                }
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int p = 0; p < 8; ++p) acc[f][p] = f32x4{0.f, 0.f, 0.f, 0.f};
            cit += gridDim.x;
            if (cit >= pl.items) break;
            tile_of(cit, bt, sp, m0, n0);
            crem = steps_of(sp);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (grp == 0) __builtin_amdgcn_s_barrier();               // pairs with group 1's last barrier
}

// ---------------------------------------------------------------------------------------------------------
namespace {
template <bool AMN, bool BMN, int EPI> int pg_go(const TgArgs& a, const PgPlan& pl, hipStream_t stream) {
    static std::atomic<unsigned long long> attr_done{0};
    if (const int rc = mis_set_dyn_lds(attr_done, reinterpret_cast<const void*>(&tg_pp_kernel<AMN, BMN, EPI>), PG_LDS, "token product")) return rc;
    const int cus = mis_persist_cus();
    hipLaunchKernelGGL((tg_pp_kernel<AMN, BMN, EPI>), dim3((unsigned)(pl.items < cus ? pl.items : cus)), dim3(512), PG_LDS, stream, a, pl);
    MIS_LAUNCH_CHECK("token product (256 x 256)");
    return MIS_OK;
}
}   // namespace

int tg_pp_launch(int a_mn, int b_mn, int epi, const TgArgs& a, float* slab, int splits, hipStream_t stream) {
    PgPlan pl;
    const long long tm = (a.M + 255) / 256, tn = (a.N + (epi == TG_GATED ? 127 : 255)) / (epi == TG_GATED ? 128 : 256), spr = (a.K + 63) / 64;
    pl.tm = (int)tm; pl.tn = (int)tn;
    pl.spr = (int)spr;
    pl.sps = (int)((spr * a.ranges + splits - 1) / splits);
    pl.splits = (int)((spr * a.ranges + pl.sps - 1) / pl.sps);          // (no part is empty)
    pl.slab = slab;
    const long long items = tm * tn * a.batches * pl.splits;
    MIS_REQUIRE(items < (1ll << 30) && spr * a.ranges < (1ll << 30), MIS_EUNSUPPORTED, "token product: %lld tiles of %lld steps are too many", items, spr * a.ranges);
    pl.items = (int)items;
    if (epi == TG_GATED) return pg_go<false, false, TG_GATED>(a, pl, stream);
    if (!a_mn && !b_mn) return pg_go<false, false, TG_LINEAR>(a, pl, stream);
    int rc;
    if (pl.splits == 1) return a_mn ? pg_go<true, true, TG_STORE>(a, pl, stream) : pg_go<false, true, TG_STORE>(a, pl, stream);
    rc = a_mn ? pg_go<true, true, TG_SLAB>(a, pl, stream) : pg_go<false, true, TG_SLAB>(a, pl, stream);
    if (rc) return rc;
    return tg_slab_sum(MIS_BF16, a, slab, pl.splits, stream);
}
