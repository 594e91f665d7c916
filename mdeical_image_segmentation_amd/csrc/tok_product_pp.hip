// Large bf16 matrix products of the token operators: a persistent 256 x 256 ping-pong kernel, all three operand layouts (tok_gemm.hpp), 16-byte aligned operands.
//
// 8 waves, 2 (m) x 4 (n), a wave owns 128 x 64 of C as 8 x 4 MFMA tiles of 16 x 16 (128 accumulator registers).  A step is 64 k: two segments of 12 fragments (24 KiB of LDS reads per
// wave and step for 64 MFMAs) - the two waves of a SIMD are one barrier apart, so that one is always inside its 32 MFMAs (512 cycles) while the other fetches fragments:
//
//      slot        0            1            2            3               4
//      group 0     R0 B(s+1)    M0           R1 A(s+2) w  M1              R0' ...      R = fragment reads, M = 32 MFMAs, every slot ends with a barrier of all 8 waves
//      group 1     M1"          R0 B(s+1)    M0           w R1 A(s+2)     M1 ...       w = wait for this wave's part of step s + 1
//
// Both operands arrive by LDS-DMA, 64 KiB a step, four instructions of 1 KiB per wave in each of its R segments: the CU's load path takes about 25 cycles for one, and a wave that
// issues into the full path stalls (two of them inside an M segment made it 800 cycles long).  B is double-buffered and fetched one step ahead, A has three buffers and is fetched two
// steps ahead (all 160 KiB of LDS); a buffer's last readers passed the barrier in front of the slot that refills it, and step s + 1 is waited for a segment before the barrier
// in front of its first read, by a count that leaves group 0's four A(s+2) in flight.  The step sequence is flat over a block's tiles (grid = number of CUs), so a tile's first steps are in flight while the tile before is finished and stored.
// LDS images and swizzles are those of tok_product.hpp with 256 rows: [row][128 B] for a k-contiguous operand, [k][512 B] for the other kind, read with the transposing ds_read_b64_tr_b16.
// Bound: per step 192 KiB of fragments leave and 64 KiB enter the LDS, 2048 cycles at its 128 B a cycle - as many as the MFMAs take, so every cycle of a segment that is neither shows.
// 8192^3 770 us, 1.43 PFLOP/s (x W^T; dz W 783, dz^T x 837); 32768 x 1024 x 8192, 16 steps a tile: 493 us, 1.11, of which 4 to 5 steps' time a tile is the store of its 128 KiB.  A wave
// tile of 128 x 128 would need a third less from the LDS, but 256 accumulators and 64 fragment registers a lane do not fit beside the addresses.
// The fragment reads and their wait are one asm statement: hipcc would put a vmcnt(0), i.e. a wait for the prefetch, in front of a plain LDS read while an LDS-DMA is in flight.

#include "conv_pp_common.hpp"
#include "dispatch_cfg.hpp"
#include "tok_epilogue.hpp"
#include "tok_product_plan.hpp"

typedef __attribute__((ext_vector_type(4))) int i32x4;

namespace {
constexpr int PG_OP = 32768;              // bytes of one operand's 64-k step
constexpr int PG_B0 = 3 * PG_OP;          // LDS: three A buffers, two B buffers
constexpr int PG_LDS = 5 * PG_OP;

// One segment's LDS traffic of a wave as one statement: 12 fragments are asked for, then (DMA) the four LDS-DMA instructions of a step - issuing them takes longer than the LDS needs
// to answer - and the fragments waited for.  One statement, because a plain LDS read beside an LDS-DMA in flight makes hipcc wait for the prefetch first, and a read whose wait stands
// elsewhere leaves the compiler free to move a register that the LDS has not written yet.
//   aA / aB: this lane's LDS address of fragment 0
struct PgDma {
    unsigned v[4];          // byte offsets of this lane (one past num_records: zeros)
    i32x4 rsrc;
    int step;               // scalar offset between the instructions
    uint32_t dst;           // LDS address of the first one; 8 KiB between them
};
#define PG_DMA(V0, V1, V2, V3, R, ST, D, T)                                                                                                   \
    "s_mov_b32 m0, %" D "\n\ts_nop 4\n\tbuffer_load_dwordx4 %" V0 ", %" R ", 0 offen lds\n\t"                                                  \
    "s_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\tbuffer_load_dwordx4 %" V1 ", %" R ", %" ST " offen lds\n\t"                                          \
    "s_add_u32 m0, m0, 0x2000\n\ts_lshl_b32 %" T ", %" ST ", 1\n\tbuffer_load_dwordx4 %" V2 ", %" R ", %" T " offen lds\n\t"                      \
    "s_add_u32 m0, m0, 0x2000\n\ts_add_u32 %" T ", %" T ", %" ST "\n\tbuffer_load_dwordx4 %" V3 ", %" R ", %" T " offen lds\n\t"

__device__ __forceinline__ void pg_read_kk(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB) {
    asm volatile(
        "ds_read_b128 %0, %13\n\t"
        "ds_read_b128 %1, %13 offset:512\n\t"
        "ds_read_b128 %2, %13 offset:4096\n\t"
        "ds_read_b128 %3, %13 offset:4608\n\t"
        "ds_read_b128 %4, %12\n\t"
        "ds_read_b128 %5, %12 offset:2048\n\t"
        "ds_read_b128 %6, %12 offset:4096\n\t"
        "ds_read_b128 %7, %12 offset:6144\n\t"
        "ds_read_b128 %8, %12 offset:8192\n\t"
        "ds_read_b128 %9, %12 offset:10240\n\t"
        "ds_read_b128 %10, %12 offset:12288\n\t"
        "ds_read_b128 %11, %12 offset:14336\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(B[0]), "=&v"(B[1]), "=&v"(B[2]), "=&v"(B[3]), "=&v"(A[0]), "=&v"(A[1]), "=&v"(A[2]), "=&v"(A[3]), "=&v"(A[4]), "=&v"(A[5]), "=&v"(A[6]), "=&v"(A[7])
        : "v"(aA), "v"(aB)
        : "memory");
}
__device__ __forceinline__ void pg_read_kk_dma(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB, const PgDma& d) {
    int t;
    asm volatile(
        "ds_read_b128 %0, %14\n\t"
        "ds_read_b128 %1, %14 offset:512\n\t"
        "ds_read_b128 %2, %14 offset:4096\n\t"
        "ds_read_b128 %3, %14 offset:4608\n\t"
        "ds_read_b128 %4, %13\n\t"
        "ds_read_b128 %5, %13 offset:2048\n\t"
        "ds_read_b128 %6, %13 offset:4096\n\t"
        "ds_read_b128 %7, %13 offset:6144\n\t"
        "ds_read_b128 %8, %13 offset:8192\n\t"
        "ds_read_b128 %9, %13 offset:10240\n\t"
        "ds_read_b128 %10, %13 offset:12288\n\t"
        "ds_read_b128 %11, %13 offset:14336\n\t"
        PG_DMA("15", "16", "17", "18", "19", "20", "21", "12")
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(B[0]), "=&v"(B[1]), "=&v"(B[2]), "=&v"(B[3]), "=&v"(A[0]), "=&v"(A[1]), "=&v"(A[2]), "=&v"(A[3]), "=&v"(A[4]), "=&v"(A[5]), "=&v"(A[6]), "=&v"(A[7]), "=&s"(t)
        : "v"(aA), "v"(aB), "v"(d.v[0]), "v"(d.v[1]), "v"(d.v[2]), "v"(d.v[3]), "s"(d.rsrc), "s"(d.step), "s"(d.dst)
        : "memory", "scc", "m0");
}
__device__ __forceinline__ u32x4 pg_join(const u32x2& lo, const u32x2& hi) { return u32x4{lo[0], lo[1], hi[0], hi[1]}; }
// B with its own index contiguous: fragment f at aB ^ (64 if f >= 2), + 8 bytes if f is odd; the second half of its k 4 rows (2048 B) further
__device__ __forceinline__ void pg_read_km(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB) {
    u32x2 b[8];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %17\n\t"
        "ds_read_b64_tr_b16 %1, %17 offset:2048\n\t"
        "ds_read_b64_tr_b16 %2, %17 offset:8\n\t"
        "ds_read_b64_tr_b16 %3, %17 offset:2056\n\t"
        "ds_read_b64_tr_b16 %4, %18\n\t"
        "ds_read_b64_tr_b16 %5, %18 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %18 offset:8\n\t"
        "ds_read_b64_tr_b16 %7, %18 offset:2056\n\t"
        "ds_read_b128 %8, %16\n\t"
        "ds_read_b128 %9, %16 offset:2048\n\t"
        "ds_read_b128 %10, %16 offset:4096\n\t"
        "ds_read_b128 %11, %16 offset:6144\n\t"
        "ds_read_b128 %12, %16 offset:8192\n\t"
        "ds_read_b128 %13, %16 offset:10240\n\t"
        "ds_read_b128 %14, %16 offset:12288\n\t"
        "ds_read_b128 %15, %16 offset:14336\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(b[4]), "=&v"(b[5]), "=&v"(b[6]), "=&v"(b[7]), "=&v"(A[0]), "=&v"(A[1]), "=&v"(A[2]), "=&v"(A[3]), "=&v"(A[4]), "=&v"(A[5]), "=&v"(A[6]), "=&v"(A[7])
        : "v"(aA), "v"(aB), "v"(aB ^ 64u)
        : "memory");
#pragma unroll
    for (int f = 0; f < 4; ++f) B[f] = pg_join(b[2 * f], b[2 * f + 1]);
}
__device__ __forceinline__ void pg_read_km_dma(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB, const PgDma& d) {
    u32x2 b[8];
    int t;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %18\n\t"
        "ds_read_b64_tr_b16 %1, %18 offset:2048\n\t"
        "ds_read_b64_tr_b16 %2, %18 offset:8\n\t"
        "ds_read_b64_tr_b16 %3, %18 offset:2056\n\t"
        "ds_read_b64_tr_b16 %4, %19\n\t"
        "ds_read_b64_tr_b16 %5, %19 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %19 offset:8\n\t"
        "ds_read_b64_tr_b16 %7, %19 offset:2056\n\t"
        "ds_read_b128 %8, %17\n\t"
        "ds_read_b128 %9, %17 offset:2048\n\t"
        "ds_read_b128 %10, %17 offset:4096\n\t"
        "ds_read_b128 %11, %17 offset:6144\n\t"
        "ds_read_b128 %12, %17 offset:8192\n\t"
        "ds_read_b128 %13, %17 offset:10240\n\t"
        "ds_read_b128 %14, %17 offset:12288\n\t"
        "ds_read_b128 %15, %17 offset:14336\n\t"
        PG_DMA("20", "21", "22", "23", "24", "25", "26", "16")
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(b[4]), "=&v"(b[5]), "=&v"(b[6]), "=&v"(b[7]), "=&v"(A[0]), "=&v"(A[1]), "=&v"(A[2]), "=&v"(A[3]), "=&v"(A[4]), "=&v"(A[5]), "=&v"(A[6]), "=&v"(A[7]), "=&s"(t)
        : "v"(aA), "v"(aB), "v"(aB ^ 64u), "v"(d.v[0]), "v"(d.v[1]), "v"(d.v[2]), "v"(d.v[3]), "s"(d.rsrc), "s"(d.step), "s"(d.dst)
        : "memory", "scc", "m0");
#pragma unroll
    for (int f = 0; f < 4; ++f) B[f] = pg_join(b[2 * f], b[2 * f + 1]);
}
// both of the other kind: A's fragment p at aA ^ (32 p).  Two statements: an asm statement holds 30 operands
__device__ __forceinline__ void pg_read_mm1(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB) {
    u32x2 b[8], a[8];
    uint32_t x;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %18\n\t"
        "ds_read_b64_tr_b16 %1, %18 offset:2048\n\t"
        "ds_read_b64_tr_b16 %2, %18 offset:8\n\t"
        "ds_read_b64_tr_b16 %3, %18 offset:2056\n\t"
        "ds_read_b64_tr_b16 %4, %19\n\t"
        "ds_read_b64_tr_b16 %5, %19 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %19 offset:8\n\t"
        "ds_read_b64_tr_b16 %7, %19 offset:2056\n\t"
        "ds_read_b64_tr_b16 %8, %17\n\t"
        "ds_read_b64_tr_b16 %9, %17 offset:2048\n\t"
        "v_xor_b32 %16, 0x20, %17\n\t"
        "ds_read_b64_tr_b16 %10, %16\n\t"
        "ds_read_b64_tr_b16 %11, %16 offset:2048\n\t"
        "v_xor_b32 %16, 0x40, %17\n\t"
        "ds_read_b64_tr_b16 %12, %16\n\t"
        "ds_read_b64_tr_b16 %13, %16 offset:2048\n\t"
        "v_xor_b32 %16, 0x60, %17\n\t"
        "ds_read_b64_tr_b16 %14, %16\n\t"
        "ds_read_b64_tr_b16 %15, %16 offset:2048\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(b[4]), "=&v"(b[5]), "=&v"(b[6]), "=&v"(b[7]), "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7]), "=&v"(x)
        : "v"(aA), "v"(aB), "v"(aB ^ 64u)
        : "memory");
#pragma unroll
    for (int f = 0; f < 4; ++f) B[f] = pg_join(b[2 * f], b[2 * f + 1]);
#pragma unroll
    for (int p = 0; p < 4; ++p) A[p] = pg_join(a[2 * p], a[2 * p + 1]);
}
__device__ __forceinline__ void pg_read_mm1_dma(u32x4 (&A)[8], u32x4 (&B)[4], uint32_t aA, uint32_t aB, const PgDma& d) {
    u32x2 b[8], a[8];
    int t;
    uint32_t x;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %19\n\t"
        "ds_read_b64_tr_b16 %1, %19 offset:2048\n\t"
        "ds_read_b64_tr_b16 %2, %19 offset:8\n\t"
        "ds_read_b64_tr_b16 %3, %19 offset:2056\n\t"
        "ds_read_b64_tr_b16 %4, %20\n\t"
        "ds_read_b64_tr_b16 %5, %20 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %20 offset:8\n\t"
        "ds_read_b64_tr_b16 %7, %20 offset:2056\n\t"
        "ds_read_b64_tr_b16 %8, %18\n\t"
        "ds_read_b64_tr_b16 %9, %18 offset:2048\n\t"
        "v_xor_b32 %16, 0x20, %18\n\t"
        "ds_read_b64_tr_b16 %10, %16\n\t"
        "ds_read_b64_tr_b16 %11, %16 offset:2048\n\t"
        "v_xor_b32 %16, 0x40, %18\n\t"
        "ds_read_b64_tr_b16 %12, %16\n\t"
        "ds_read_b64_tr_b16 %13, %16 offset:2048\n\t"
        "v_xor_b32 %16, 0x60, %18\n\t"
        "ds_read_b64_tr_b16 %14, %16\n\t"
        "ds_read_b64_tr_b16 %15, %16 offset:2048\n\t"
        PG_DMA("21", "22", "23", "24", "25", "26", "27", "17")
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(b[4]), "=&v"(b[5]), "=&v"(b[6]), "=&v"(b[7]), "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7]), "=&v"(x), "=&s"(t)
        : "v"(aA), "v"(aB), "v"(aB ^ 64u), "v"(d.v[0]), "v"(d.v[1]), "v"(d.v[2]), "v"(d.v[3]), "s"(d.rsrc), "s"(d.step), "s"(d.dst)
        : "memory", "scc", "m0");
#pragma unroll
    for (int f = 0; f < 4; ++f) B[f] = pg_join(b[2 * f], b[2 * f + 1]);
#pragma unroll
    for (int p = 0; p < 4; ++p) A[p] = pg_join(a[2 * p], a[2 * p + 1]);
}
__device__ __forceinline__ void pg_read_mm2(u32x4 (&A)[8], uint32_t aA) {
    u32x2 a[8];
    uint32_t x;
    asm volatile(
        "v_xor_b32 %8, 0x80, %9\n\t"
        "ds_read_b64_tr_b16 %0, %8\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:2048\n\t"
        "v_xor_b32 %8, 0xa0, %9\n\t"
        "ds_read_b64_tr_b16 %2, %8\n\t"
        "ds_read_b64_tr_b16 %3, %8 offset:2048\n\t"
        "v_xor_b32 %8, 0xc0, %9\n\t"
        "ds_read_b64_tr_b16 %4, %8\n\t"
        "ds_read_b64_tr_b16 %5, %8 offset:2048\n\t"
        "v_xor_b32 %8, 0xe0, %9\n\t"
        "ds_read_b64_tr_b16 %6, %8\n\t"
        "ds_read_b64_tr_b16 %7, %8 offset:2048\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7]), "=&v"(x)
        : "v"(aA)
        : "memory");
#pragma unroll
    for (int p = 0; p < 4; ++p) A[4 + p] = pg_join(a[2 * p], a[2 * p + 1]);
}

// Where this lane's 16 bytes of an operand's DMA instructions lie, relative to the step's first element
struct PgLane {
    unsigned v0;            // byte offset in the wave's first instruction
    unsigned jstep;         // ... and between its four instructions: 64 rows (gated B: 32 columns) or 16 k further
    int row;                // k contiguous: row of the first instruction; else first column of the chunk
    int k;                  // k contiguous: first k of the chunk; else k row of the first instruction
};
// one operand's 64-k step: its first element, and this lane's four byte offsets.  Valid lanes are inside the operand by construction; a lane that has to read zeros (behind the last
// row or k) carries an offset past num_records.
struct PgStep {
    const char* base;
    unsigned v[4];
};
template <bool MN, int RSTEP> __device__ __forceinline__ void pg_mask(const PgLane& l, PgStep& s, int left, int rows) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool ok = MN ? (l.k + 16 * j < left && l.row < rows) : (l.k < left && l.row + RSTEP * j < rows);
        s.v[j] = ok ? l.v0 : (unsigned)PP_OOB;
    }
}
__device__ __forceinline__ PgDma pg_dma(const PgLane& l, const PgStep& s, uint32_t dst) {
    const uintptr_t b = (uintptr_t)s.base;
    return PgDma{{s.v[0], s.v[1], s.v[2], s.v[3]}, i32x4{(int)(uint32_t)b, (int)(b >> 32), 0x7fffffff, 0x00020000}, (int)l.jstep, dst};          // raw buffer, stride 0
}
__device__ __forceinline__ void pg_issue(const PgDma& d) {
    int t;
    asm volatile(PG_DMA("1", "2", "3", "4", "5", "6", "7", "0") "" : "=&s"(t) : "v"(d.v[0]), "v"(d.v[1]), "v"(d.v[2]), "v"(d.v[3]), "s"(d.rsrc), "s"(d.step), "s"(d.dst) : "memory", "scc", "m0");
}
}   // namespace

template <bool AMN, bool BMN, int EPI, int ACT>
__global__ __launch_bounds__(512, 2) void tg_pp_kernel(const TgArgs a, const TpPlan pl) {
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
    if constexpr (!BMN) fB = wn * 8192 + (8 * (li >> 2) + (li & 3)) * 128 + ((lg ^ (((li >> 1) & 1) | ((li >> 2) << 1))) << 4);
    else fB = (8 * lg + (li >> 2)) * 512 + (((wn * 4 + ((li & 3) >> 1)) ^ ((li >> 2) << 1)) << 5) + 16 * (li & 1);

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
    auto tile_of = [&](int it) __attribute__((always_inline)) {
        TpItem w;
        const int t = it % tiles, bs = it / tiles;
        w.sp = bs % pl.splits;
        w.bt = bs / pl.splits;
        const int band = t / (4 * pl.tn), in = t - band * 4 * pl.tn;
        const int h = pl.tm - band * 4 < 4 ? pl.tm - band * 4 : 4;
        const int c = in / h;
        w.m0 = (long long)(band * 4 + in - c * h) * 256;
        w.n0 = (long long)c * BN;
        return w;
    };
    auto steps_of = [&](int sp) __attribute__((always_inline)) {
        const int s0 = sp * pl.sps;
        return nsteps_all - s0 < pl.sps ? nsteps_all - s0 : pl.sps;
    };

    // ---- load cursor: `na` is the step whose A is issued next, `nb` the one whose B is (the step before, once the pipeline runs) ----
    int lit = first, lrem = 0, krem = 0;                      // item; its steps, and k of its range, from the cursor's step on
    int rows_a = 0, rows_b = 0;                               // rows and columns of its tile that exist
    PgStep na, nb, nb1;                                       // nb1: B of na's step
    int va = 1, vb = 1;                                       // whether na / nb is a step of this block
    const long long step_a = AMN ? 128 * a.a.ld : 128, step_b = BMN ? 128 * a.b.ld : 128;
    auto masks = [&]() __attribute__((always_inline)) {
        const int left = krem < 64 ? krem : 64;
        pg_mask<AMN, 64>(la, na, left, rows_a);
        pg_mask<BMN, BROWS>(lb, nb1, left, rows_b);
    };
    // (tile, k part) of item lit at step `at` of its product -> na, nb1
    auto place = [&](long long m0, long long n0, int bt, int at) __attribute__((always_inline)) {
        const int range = at >= pl.spr ? 1 : 0, ks = at - range * pl.spr;
        // (p + s (p2 - p), not s ? p2 : p: hipcc turns that into an indexed load from a scratch copy of the arguments)
        const char* const pa = (const char*)a.a.p + (long long)(EPI == TG_GATED ? 0 : bt | range) * ((const char*)a.a.p2 - (const char*)a.a.p);
        const char* const pb = (const char*)a.b.p + (long long)(EPI == TG_GATED ? (wave >> 2) : bt | range) * ((const char*)a.b.p2 - (const char*)a.b.p);
        na.base = pa + (AMN ? m0 : m0 * a.a.ld) * 2 + ks * step_a;
        nb1.base = pb + (BMN ? n0 : n0 * a.b.ld) * 2 + ks * step_b;
        krem = (int)a.K - ks * 64;
        rows_a = a.M - m0 < 256 ? (int)(a.M - m0) : 256;
        rows_b = a.N - n0 < BN ? (int)(a.N - n0) : BN;
        masks();
    };
    // the first step of item lit, or (second) of its second range
    auto load_tile = [&](bool second) __attribute__((always_inline)) {
        const TpItem w = tile_of(lit);
        if (!second) lrem = steps_of(w.sp);
        place(w.m0, w.n0, w.bt, second ? pl.spr : w.sp * pl.sps);
    };
    // A of the cursor's step is issued: its B is next, and A of the step behind it.  One untaken branch but at the ends of ranges and tiles and on the step behind one (when B takes over
    // the masks that A got): a chain of taken branches here cost 390 cycles a step, 8192^3 789 us instead of 759.
    int changed = 0;
    auto advance = [&]() __attribute__((always_inline)) {
        const int rare = changed | (va & ((lrem == 1 ? 1 : 0) | (krem < 128 ? 1 : 0)));
        nb.base = nb1.base;
        vb = va;
        na.base += step_a;
        nb1.base += step_b;
        krem -= 64;
        lrem -= 1;
        if (__builtin_expect(rare, 0)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) nb.v[j] = nb1.v[j];
            changed = 0;
            if (va && (lrem == 0 || krem < 64)) {
                if (lrem == 0) {
                    lit += gridDim.x;
                    va = __builtin_amdgcn_readfirstlane(lit < pl.items ? 1 : 0);
                }
                if (lrem != 0 && krem > 0) masks();           // the last, short step of a range
                else if (va) load_tile(lrem != 0);
                changed = 1;
            }
        }
    };
    load_tile(false);

    f32x4 acc[4][8];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int p = 0; p < 8; ++p) acc[f][p] = f32x4{0.f, 0.f, 0.f, 0.f};

    // LDS addresses of the current step's buffers, and of where B(s + 1) and A(s + 2) of this wave go
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem, ldsB = lds0 + PG_B0;
    uint32_t curA = lds0, curB = ldsB, dstA = lds0 + 2 * PG_OP + wave * 1024, dstB = ldsB + PG_OP + wave * 1024;
    pg_issue(pg_dma(la, na, lds0 + wave * 1024));
    changed = 1;
    advance();
    pg_issue(pg_dma(lb, nb, ldsB + wave * 1024));
    if (va) pg_issue(pg_dma(la, na, lds0 + PG_OP + wave * 1024));          // A of step 1
    advance();                                                // nb: B of step 1, na: A of step 2
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_sleep(4);                              // 256 cycles between the first steps' arrival and the barrier behind which other waves read them (see retire)
    __syncthreads();
    if (grp == 1) __builtin_amdgcn_s_barrier();               // the stagger
    __builtin_amdgcn_sched_barrier(0);

    int cit = first;
    TpItem ct = tile_of(cit);
    int crem = steps_of(ct.sp);

    u32x4 fa[8], fb[4];
    // the fragments of half kk; with `dma` also this segment's part of the prefetch: B of step s + 1 (half 0), A of step s + 2 (half 1)
    auto read = [&](int kk, int dma) __attribute__((always_inline)) {
        // k-contiguous: the second half of the step is 64 bytes further in the row, i.e. chunk position ^ 4; else 32 k rows further
        const uint32_t xa = curA + (AMN ? fA + kk * 16384 : fA ^ (kk * 64));
        const uint32_t xb = curB + (BMN ? fB + kk * 16384 : fB ^ (kk * 64));
        if (dma) {
            const PgDma d = kk == 0 ? pg_dma(lb, nb, dstB) : pg_dma(la, na, dstA);
            if constexpr (!AMN && !BMN) pg_read_kk_dma(fa, fb, xa, xb, d);
            else if constexpr (!AMN) pg_read_km_dma(fa, fb, xa, xb, d);
            else pg_read_mm1_dma(fa, fb, xa, xb, d);
        } else {
            if constexpr (!AMN && !BMN) pg_read_kk(fa, fb, xa, xb);
            else if constexpr (!AMN) pg_read_km(fa, fb, xa, xb);
            else pg_read_mm1(fa, fb, xa, xb);
        }
        if constexpr (AMN) pg_read_mm2(fa, xa);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto mma = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int p = 0; p < 8; ++p) mma_b128<T>(acc[f][p], fb[f], fa[p]);
#pragma unroll
        for (int i = 0; i < 16; ++i) {                        // two MFMAs, then what fits beside them
            __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x6, 2, 0);
        }
    };
    auto barrier = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    // Step s + 1 is complete in this wave's part once at most the four A(s + 2) just issued are in flight.  Both groups wait for it a whole segment before the barrier in front of its first
    // read (slot 4), not right at that barrier: a read that starts within a few dozen cycles of another wave's vmcnt wait can still see the old contents of the last bytes of its LDS-DMA.
    // Between the wait and that barrier lie group 0's 32 MFMAs (slot 3) and group 1's 12 fragment reads with their own wait (slot 3); scripts/codegen_guard.py pins both.
    auto retire = [&](int inflight) __attribute__((always_inline)) {
        if (inflight) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };

#pragma unroll 1
    while (true) {
        // ---- segment 0 ----
        read(0, vb);
        barrier();
        __builtin_amdgcn_s_setprio(1);
        mma();
        __builtin_amdgcn_s_setprio(0);
        barrier();
        // ---- segment 1 ----
        if (grp == 1) retire(0);                              // (its B(s + 1) is the youngest: A(s + 2) goes out with the reads below)
        read(1, va);
        if (grp == 0) retire(va);
        barrier();
        __builtin_amdgcn_s_setprio(1);
        curA = curA == lds0 + 2 * PG_OP ? lds0 : curA + PG_OP;
        dstA = curA == lds0 ? lds0 + 2 * PG_OP + wave * 1024 : curA - PG_OP + wave * 1024;
        dstB = curB + wave * 1024;
        curB = ldsB + PG_OP - (curB - ldsB);
        mma();
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        advance();
        barrier();
        if (--crem == 0) {
            // ---- the tile is complete: group 0 waits for group 1's last M, and both store at once (one after the other they would leave each SIMD to one wave's dependent VALU
            // instructions: 32768 x 1024 x 2 x 4096 with SiLU and half the bytes kept 600 -> 536 us; with all of them 616, with none 454) ----
            if (grp == 0) barrier();
            if constexpr (EPI == TG_GATED) {
                const TgGatedRow<T, ACT> row(a, ct.n0 + wn * 32 + 8 * lg);
                if (row.nv > 0) {
#pragma unroll
                    for (int p = 0; p < 8; ++p) {
                        const long long m = ct.m0 + wm * 128 + 16 * p + li;
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
                    const long long n = ct.n0 + wn * 64 + 32 * h + 8 * lg;
                    const TgLinearRow<T, ACT> row(a, tg_out(a, ct.bt), n, EPI == TG_LINEAR);
                    float* const sl = pl.slab + (long long)(ct.bt * pl.splits + ct.sp) * a.M * a.N + n;
                    if (row.nv > 0) {
#pragma unroll
                        for (int p = 0; p < 8; ++p) {
                            const long long m = ct.m0 + wm * 128 + 16 * p + li;
                            float v[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = acc[2 * h + (j >> 2)][p][j & 3];
                            if (m < a.M) {
                                if constexpr (EPI == TG_LINEAR) row(m, v);
                                else if constexpr (EPI == TG_STORE) row.store(m, v);
                                else tok_stn<float>(sl + m * a.N, v, row.nv);
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
            ct = tile_of(cit);
            crem = steps_of(ct.sp);
            if (grp == 1) barrier();                          // the stagger again
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
namespace {
template <bool AMN, bool BMN, int EPI, int ACT = MIS_ACT_NONE> int pg_go(const TgArgs& a, const TpPlan& pl, hipStream_t stream) {
    static std::atomic<unsigned long long> attr_done{0};
    if (const int rc = mis_set_dyn_lds(attr_done, reinterpret_cast<const void*>(&tg_pp_kernel<AMN, BMN, EPI, ACT>), PG_LDS, "token product")) return rc;
    const int cus = mis_persist_cus();
    hipLaunchKernelGGL((tg_pp_kernel<AMN, BMN, EPI, ACT>), dim3((unsigned)(pl.items < cus ? pl.items : cus)), dim3(512), PG_LDS, stream, a, pl);
    MIS_LAUNCH_CHECK("token product (256 x 256)");
    return MIS_OK;
}
template <int EPI> int pg_act(const TgArgs& a, const TpPlan& pl, hipStream_t stream) {
    switch (a.act) {
        case MIS_ACT_RELU: return pg_go<false, false, EPI, MIS_ACT_RELU>(a, pl, stream);
        case MIS_ACT_GELU: return pg_go<false, false, EPI, MIS_ACT_GELU>(a, pl, stream);
        case MIS_ACT_GELU_TANH: return pg_go<false, false, EPI, MIS_ACT_GELU_TANH>(a, pl, stream);
        case MIS_ACT_SILU: return pg_go<false, false, EPI, MIS_ACT_SILU>(a, pl, stream);
        case MIS_ACT_SIGMOID: return pg_go<false, false, EPI, MIS_ACT_SIGMOID>(a, pl, stream);
        default: return pg_go<false, false, EPI, MIS_ACT_NONE>(a, pl, stream);
    }
}
}   // namespace

int tok_product_bf16_256(int a_mn, int b_mn, int epi, const TgArgs& a, const TpPlan& pl, hipStream_t stream) {
    if (epi == TG_GATED) return pg_act<TG_GATED>(a, pl, stream);
    if (epi == TG_LINEAR) return pg_act<TG_LINEAR>(a, pl, stream);
    if (!b_mn) return pg_go<false, false, TG_SLAB>(a, pl, stream);
    if (epi == TG_STORE) return a_mn ? pg_go<true, true, TG_STORE>(a, pl, stream) : pg_go<false, true, TG_STORE>(a, pl, stream);
    return a_mn ? pg_go<true, true, TG_SLAB>(a, pl, stream) : pg_go<false, true, TG_SLAB>(a, pl, stream);
}
