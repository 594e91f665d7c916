// Dispatch of the token products (tok_gemm.hpp): tile size, parts along k, and the sum of the parts.
#include "dispatch_cfg.hpp"
#include "tok_epilogue.hpp"
#include "tok_product_plan.hpp"

// A product's k parts added in their order, then its epilogue: a rounded store (batch 1 goes to y2), bias + activation + residual, or act(batch 0) * batch 1
template <typename T, int EPI> __device__ __forceinline__ void tg_slab_run(const TgArgs& a, const float* __restrict__ slab, int splits, long long id) {
    const long long per = (a.N + 7) >> 3;
    const long long row = id / per, n = (id - row * per) * 8;
    const int nv = a.N - n >= 8 ? 8 : (int)(a.N - n);
    const int bt = EPI == TG_STORE && row >= a.M ? 1 : 0;
    const long long m = row - bt * a.M;
    auto sum = [&](int batch, float (&v)[8]) __attribute__((always_inline)) {
        const float* p = slab + ((long long)batch * splits * a.M + m) * a.N + n;
        tok_ldn<float>(p, v, nv);
        for (int s = 1; s < splits; ++s) {
            float t[8];
            tok_ldn<float>(p + (long long)s * a.M * a.N, t, nv);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += t[j];
        }
    };
    float v[8];
    sum(bt, v);
    if constexpr (EPI == TG_STORE) {
        tok_stn<T>(reinterpret_cast<T*>(tg_out(a, bt)) + m * a.ldy + n, v, nv);
    } else if constexpr (EPI == TG_LINEAR) {
        const TgLinearRow<T> r(a, a.y, n, true);
        r(m, v);
    } else {
        float u[8];
        sum(1, u);
        const TgGatedRow<T> r(a, n);
        r(m, v, u);
    }
}
template <typename T, int EPI> __global__ __launch_bounds__(256) void tg_slab_kernel(const TgSum s) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id < s.runs) tg_slab_run<T, EPI>(s.a, s.slab, s.splits, id);
}
// two products' sums: the first nb0 blocks add s, the others t
template <typename T> __global__ __launch_bounds__(256) void tg_slab2_kernel(const TgSum s, const TgSum t, unsigned nb0) {
    if (blockIdx.x < nb0) {
        const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
        if (id < s.runs) tg_slab_run<T, TG_STORE>(s.a, s.slab, s.splits, id);
    } else {
        const long long id = (long long)(blockIdx.x - nb0) * 256 + threadIdx.x;
        if (id < t.runs) tg_slab_run<T, TG_STORE>(t.a, t.slab, t.splits, id);
    }
}

namespace {
template <typename T> void tg_slab_go(int epi, unsigned blocks, const TgSum& s, hipStream_t stream) {
    if (epi == TG_STORE) hipLaunchKernelGGL((tg_slab_kernel<T, TG_STORE>), dim3(blocks), dim3(256), 0, stream, s);
    else if (epi == TG_LINEAR) hipLaunchKernelGGL((tg_slab_kernel<T, TG_LINEAR>), dim3(blocks), dim3(256), 0, stream, s);
    else hipLaunchKernelGGL((tg_slab_kernel<T, TG_GATED>), dim3(blocks), dim3(256), 0, stream, s);
}
int tg_slab_sum(int dtype, int epi, const TgSum& s, hipStream_t stream) {
    const long long n = (s.runs + 255) / 256;
    MIS_REQUIRE(n < TOK_BLOCKS, MIS_EUNSUPPORTED, "token product: the grid is too large");
    if (dtype == MIS_BF16) tg_slab_go<__bf16>(epi, (unsigned)n, s, stream);
    else tg_slab_go<float>(epi, (unsigned)n, s, stream);
    MIS_LAUNCH_CHECK("token product (sum of k parts)");
    return MIS_OK;
}
}   // namespace

int tg_sums(int dtype, const TgSum& s, const TgSum& t, hipStream_t stream) {
    if (s.slab == nullptr && t.slab == nullptr) return MIS_OK;
    if (s.slab == nullptr || t.slab == nullptr) return tg_slab_sum(dtype, TG_STORE, s.slab != nullptr ? s : t, stream);
    const long long n0 = (s.runs + 255) / 256, n1 = (t.runs + 255) / 256;
    MIS_REQUIRE(n0 + n1 < TOK_BLOCKS, MIS_EUNSUPPORTED, "token product: the grid is too large");
    if (dtype == MIS_BF16) hipLaunchKernelGGL(tg_slab2_kernel<__bf16>, dim3((unsigned)(n0 + n1)), dim3(256), 0, stream, s, t, (unsigned)n0);
    else hipLaunchKernelGGL(tg_slab2_kernel<float>, dim3((unsigned)(n0 + n1)), dim3(256), 0, stream, s, t, (unsigned)n0);
    MIS_LAUNCH_CHECK("token product (sums of k parts)");
    return MIS_OK;
}

namespace {
// How a product is cut: the cheapest of the tiles and numbers of k parts by this model.  A 64-k step of the blocks that a CU holds takes (us; blocks per CU: 1 .. what fits)
//      bf16   256 x 256  1.2 (few CUs at work) to 1.5     128 x 128  0.75, 1.15    64 x 64  0.45, 0.6, 0.7, 0.85     gated 64 x (64 + 64)  0.6, 0.9, 1.2
//      f32                                                128 x 128  4.1, 6.9      64 x 64  1.6, 2.4, 3.2, 4.0       gated 64 x (64 + 64)  2.4, 3.9, 5.4
// a tile's start and epilogue as much as 3 (256: 5) steps, a cut along k 5 us and its slab's write and read, mostly in the caches, at 7 TB/s.  M x K x N, us, each tile at its best number
// of parts (* the model's choice):
//                                       256      128       64                                          256      128       64
//      512 x 512 x 512       x W^T       17       11     *8.6      2048 x 2048 x 2048       dz W       40      *27       33
//      1024 x 4096 x 1024    x W^T       32      *24       25      4096 x 4096 x 1024       dz W      *33       42       63
//      2048 x 2048 x 2048    x W^T       44      *27       31      8192 x 1024 x 4096       dz^T x    *76       88      118
//      8192 x 1024 x 4096    x W^T      *65       82      119      8192 x 1024 x 4096       gated    *112      148      175
//      8192 x 2048 x 8192    x W^T     *214      294      440      f32 8192 x 1024 x 4096   x W^T       -     *510      527
// A forward product in parts (its epilogue then runs where they are added), us against one piece: 128 x 4096 x 1024 bf16 14 / 29, 128 x 8192 x 8192 38 / 64, f32 512 x 4096 x 1024 47 / 105.
struct TgCut {
    int tile;               // 256, 128 or 64 rows
    int splits;
    double us;
};
TgCut tg_cut_one(int dtype, int tile, bool may_split, long long M, long long N, long long K, int ranges, int batches, bool gated) {
    const int cols = gated ? (tile == 256 ? 128 : 64) : tile;
    const long long items = ((M + tile - 1) / tile) * ((N + cols - 1) / cols) * batches, steps = ((K + 63) / 64) * ranges;
    if (const int forced = mis_sw(SW_TOK_SPLITS); may_split && forced > 0) return TgCut{tile, (int)(forced < steps ? forced : steps), 0.0};
    const bool f32 = dtype == MIS_F32;
    const int fit = tile == 256 ? 1 : tile == 128 ? 2 : gated ? 3 : 4;          // blocks that a CU holds
    const double one = tile == 128 ? (f32 ? 1.3 : 0.35) : gated ? (f32 ? 0.9 : 0.28) : (f32 ? 0.75 : 0.3), more = tile == 128 ? (f32 ? 2.8 : 0.4) : gated ? (f32 ? 1.5 : 0.31) : (f32 ? 0.82 : 0.14);
    TgCut best{tile, 1, 1e30};
    for (int s = 1; s <= (may_split ? 32 : 1) && (s == 1 || steps / s >= 4); ++s) {
        const long long n = items * s, per = (n + 255) / 256;          // (256 CUs)
        const double step = tile == 256 ? 1.2 + 0.3 * (n < 256 ? n / 256.0 : 1.0) : one + more * (double)(per < fit ? per : fit);
        double us = (double)((n + 256 * fit - 1) / (256 * fit)) * ((double)((steps + s - 1) / s) + (tile == 256 ? 5.0 : 3.0)) * step;
        if (s > 1) us += 5.0 + 8.0 * s * (double)M * (double)N * batches / 7e6;
        if (us < best.us * 0.97) best = TgCut{tile, s, us};
    }
    return best;
}
TgCut tg_cut(int dtype, bool aligned, bool may_split, long long M, long long N, long long K, int ranges, int batches, bool gated) {
    const int forced = mis_sw(SW_TOK_TILE);          // 1: 128, 2: 256 wherever the operands allow, 3: 64
    const bool big_ok = dtype == MIS_BF16 && aligned;
    if (forced == 1 || forced == 3 || (forced == 2 && big_ok)) return tg_cut_one(dtype, forced == 1 ? 128 : forced == 2 ? 256 : 64, may_split, M, N, K, ranges, batches, gated);
    TgCut best = tg_cut_one(dtype, 128, may_split, M, N, K, ranges, batches, gated);
    const TgCut small = tg_cut_one(dtype, 64, may_split, M, N, K, ranges, batches, gated);
    if (small.us < best.us) best = small;
    if (big_ok) {
        const TgCut big = tg_cut_one(dtype, 256, may_split, M, N, K, ranges, batches, gated);
        if (big.us <= best.us * 1.13) best = big;          // (half the traffic from the L2: 4096 x 4096 x 1024 dz^T x, two parts, 51 us against 61 where the model sees 56 and 50)
    }
    return best;
}
// 16-byte chunks from 16-byte addresses and 32-bit offsets inside a tile; a k-contiguous operand's k, the other kind's own index must be whole chunks or padded to them
bool tg_aligned(int dtype, const TgArgs& a, int a_mn, int b_mn) {
    const long long es = dtype == MIS_BF16 ? 2 : 4, epc = 16 / es;
    auto ok = [&](const TgOperand& o, int mn, long long I) {
        return ((uintptr_t)o.p | (uintptr_t)o.p2 | (size_t)(o.ld * es)) % 16 == 0 && o.ld <= (1 << 20) && (o.padded || (mn ? I : a.K) % epc == 0);
    };
    return ok(a.a, a_mn, a.M) && ok(a.b, b_mn, a.N);
}
}   // namespace

namespace {
// a forward product: in one piece with its epilogue, or - few tiles and a long k - its plain products in parts, with the epilogue where they are added
TgCut tg_cut_of(int dtype, bool aligned, int epi, bool slab, long long M, long long N, long long K, int ranges, int batches) {
    if (epi == TG_STORE) return tg_cut(dtype, aligned, true, M, N, K, ranges, batches, false);
    const TgCut whole = tg_cut(dtype, aligned, false, M, N, K, 1, 1, epi == TG_GATED);
    if (!slab) return whole;
    const TgCut parts = tg_cut(dtype, aligned, true, M, N, K, 1, epi == TG_GATED ? 2 : 1, false);
    return parts.splits > 1 && parts.us < 0.9 * whole.us ? parts : whole;
}
// (the weights' kernel gives every 16 or 32 columns a block: up to 2^29 columns its grid holds them)
bool tg_few_rows(int epi, long long M, long long N) { return epi != TG_STORE && M <= 32 && N <= (1ll << 29) && mis_sw(SW_TOK_TILE) == 0; }
}   // namespace

size_t tg_slab_bytes(int dtype, int epi, long long M, long long N, long long K, int ranges, int batches) {
    if (M == 0 || tg_few_rows(epi, M, N)) return 0;
    size_t most = 0;
    for (int al = 0; al < 2; ++al) {
        const TgCut c = tg_cut_of(dtype, al == 1, epi, true, M, N, K, ranges, batches);
        const size_t n = c.splits > 1 ? tok_align((size_t)c.splits * (epi == TG_GATED ? 2 : batches) * M * N * 4) : 0;
        if (n > most) most = n;
    }
    return most;
}

int tg_launch(int dtype, int a_mn, int b_mn, int epi_, const TgArgs& args, float* slab, hipStream_t stream, TgSum* later) {
    const bool al = tg_aligned(dtype, args, a_mn, b_mn);
    if (tg_few_rows(epi_, args.M, args.N)) return tok_product_skinny(dtype, epi_, args, al, stream);
    const TgCut c = tg_cut_of(dtype, al, epi_, slab != nullptr, args.M, args.N, args.K, args.ranges, args.batches);
    TgArgs a = args;
    if (epi_ == TG_GATED && c.splits > 1) a.batches = 2;
    const int epi = c.splits > 1 ? TG_SLAB : epi_;
    const long long T = c.tile, BN = epi == TG_GATED ? (T == 256 ? 128 : 64) : T, ck = dtype == MIS_BF16 ? 64 : 32;
    const long long tm = (a.M + T - 1) / T, tn = (a.N + BN - 1) / BN, spr = (a.K + ck - 1) / ck;
    MIS_REQUIRE(tm < (1ll << 26) && tn < (1ll << 26) && spr < (1ll << 28) && tm * tn * a.batches * c.splits < (1ll << 30), MIS_EUNSUPPORTED,
                "token product: %lld x %lld tiles of %lld steps are too many", tm, tn, spr);
    TpPlan pl;
    pl.tm = (int)tm; pl.tn = (int)tn;
    pl.spr = (int)spr;
    pl.sps = (int)((spr * a.ranges + c.splits - 1) / c.splits);
    pl.splits = (int)((spr * a.ranges + pl.sps - 1) / pl.sps);          // (no part is empty)
    pl.slab = slab;
    pl.items = (int)(tm * tn * a.batches * pl.splits);
    static int (*const kernels[2][2][2])(int, int, int, const TgArgs&, const TpPlan&, hipStream_t) = {          // [f32][64][any address]
        {{tok_product_bf16_128, tok_product_bf16_128_any}, {tok_product_bf16_64, tok_product_bf16_64_any}},
        {{tok_product_f32_128, tok_product_f32_128_any}, {tok_product_f32_64, tok_product_f32_64_any}}};
    auto* const go = T == 256 ? tok_product_bf16_256 : kernels[dtype == MIS_F32][T == 64][!al];
    if (const int rc = go(a_mn, b_mn, epi, a, pl, stream)) return rc;
    if (epi != TG_SLAB) return MIS_OK;
    const TgSum sum{a, slab, pl.splits, a.M * ((a.N + 7) / 8) * (epi_ == TG_STORE ? a.batches : 1)};
    if (later == nullptr) return tg_slab_sum(dtype, epi_, sum, stream);
    *later = sum;
    return MIS_OK;
}
