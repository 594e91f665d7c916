// Matrix product of the token operators, any shape / stride / alignment: C[m][n] = sum_k A(m, k) B(n, k).
//
// A block of 4 waves owns 128 x 128 of C (gated: 128 rows x 64 columns of h = 64 gate + 64 up columns, side by side in each wave so that the product act(g) u stays in
// registers); a wave 64 x 64 as 4 x 4 MFMA tiles of 16 x 16.  One K step = 128 bytes of k per row (64 bf16 / 32 f32): global -> registers one step ahead -> LDS -> fragments.
// B(n) feeds the MFMA's row side, A(m) its column side: a lane then holds runs of 8 consecutive n of one m, and bias, residual and stores are 16 bytes wide.
//   LDS image, k contiguous:   [row][128 B], 16-byte chunks at position c ^ key(row): a fragment read touches each bank once
//   LDS image, own index cont.: [k][128 elements]; bf16 fragments by the transposing read (16 lanes: 4 k x 4 runs of 4), f32 ones by plain 16-byte reads, which give one k of four
//                              MFMA tiles (tile v then holds the indices 4 r + v)
// Sums are f32 (MFMA accumulators); k order inside a step is the same for both operands, which is all the sum needs.
#include "dispatch_cfg.hpp"
#include "tok_epilogue.hpp"

namespace {
typedef __attribute__((address_space(3))) s16x4 tg_lds_s16x4;

template <typename T> struct TgFrag { u32x4 v[2]; };      // one operand tile of 16 x (2 MFMA "b128 steps")

constexpr int TG_TILE = 16384;                             // bytes of an operand tile in LDS: 128 x 128 B

template <typename T, bool AL> __device__ __forceinline__ u32x4 tg_chunk(const T* p, long long n) {
    constexpr int EPC = Tr<T>::EPC;
    if (n >= EPC) {
        if constexpr (AL) return *reinterpret_cast<const u32x4*>(p);
        else return tok_ld16<T>(p);
    }
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n > 0) {
        float f[EPC];
#pragma unroll
        for (int i = 0; i < EPC; ++i) f[i] = i < n ? ld_elem<T>(p + i) : 0.f;
        v = pack_chunk<T>(f);
    }
    return v;
}
// swizzle keys.  Rows of a fragment: A side 16 p + li, B side 32 (f >> 1) + 8 (li >> 2) + 4 (f & 1) + (li & 3)
template <bool B> __device__ __forceinline__ int tg_key(int row) {
    return B ? (((row >> 1) & 1) | (((row >> 3) & 3) << 1)) : ((row >> 1) & 7);
}
// 32-byte position of a [k][i] bf16 row.  A side: a group of 16 lanes reads 32 bytes of 4 rows; B side: 8 of every 16 bytes of a 64-byte run of 4 rows
template <bool B> __device__ __forceinline__ int tg_pos32(int c32, int k) {
    return B ? (c32 ^ ((k & 3) << 1)) : (c32 ^ ((k & 3) | (((k >> 3) & 1) << 2)));
}

// this thread's 4 chunks of one operand's K step [k0, k0 + CK) -> registers
template <typename T, bool MN, bool B, int EPI, bool AL>
__device__ __forceinline__ void tg_load(u32x4 (&r)[4], const void* q, const TgOperand& o, long long i0, long long I, long long k0, long long K) {
    constexpr int EPC = Tr<T>::EPC;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int id = (int)threadIdx.x + 256 * j;
        if constexpr (!MN) {
            const int row = id >> 3, c = id & 7;
            const long long k = k0 + c * EPC;
            const void* p = q;
            long long i;
            if constexpr (B && EPI == TG_GATED) {
                const int w = row >> 6, rr = row & 63;                 // rows 0..31 of a wave: gate, 32..63: the same columns of up
                p = rr < 32 ? o.p : o.p2;
                i = i0 + w * 32 + (rr & 31);
            } else {
                i = i0 + row;
            }
            r[j] = tg_chunk<T, AL>(reinterpret_cast<const T*>(p) + i * o.ld + k, i < I ? K - k : 0);
        } else {
            constexpr int CPR = 128 / EPC;                             // chunks per k row
            const int kr = id / CPR, c = id % CPR;
            const long long k = k0 + kr, i = i0 + c * EPC;
            r[j] = tg_chunk<T, AL>(reinterpret_cast<const T*>(q) + k * o.ld + i, k < K ? I - i : 0);
        }
    }
}
template <typename T, bool MN, bool B> __device__ __forceinline__ void tg_store(char* lds, const u32x4 (&r)[4]) {
    constexpr int EPC = Tr<T>::EPC;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int id = (int)threadIdx.x + 256 * j;
        int off;
        if constexpr (!MN) {
            const int row = id >> 3, c = id & 7;
            off = row * 128 + ((c ^ tg_key<B>(row)) << 4);
        } else if constexpr (sizeof(T) == 2) {
            const int k = id >> 4, c = id & 15;
            off = k * 256 + (tg_pos32<B>(c >> 1, k) << 5) + ((c & 1) << 4);
        } else {
            const int k = id >> 5, c = id & 31;
            off = k * 512 + c * 16;
        }
        lds_write_b128(lds, off, r[j]);
    }
}
// the 4 fragments of a wave's 64 rows (first row w * 64) for b128 step kk
template <typename T, bool MN, bool B> __device__ __forceinline__ void tg_frags(u32x4 (&v)[4], const char* lds, int w, int kk) {
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    if constexpr (!MN) {
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int row = w * 64 + (B ? 32 * (f >> 1) + 8 * (li >> 2) + 4 * (f & 1) + (li & 3) : 16 * f + li);
            v[f] = lds_read_b128(lds, row * 128 + (((kk * 4 + lg) ^ tg_key<B>(row)) << 4));
        }
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int i = w * 64 + (B ? 32 * (f >> 1) + 8 * (li & 3) + 4 * (f & 1) : 16 * f + 4 * (li & 3));
            s16x4 h[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = kk * 32 + 8 * lg + 4 * s + (li >> 2);
                const uint32_t at = (uint32_t)(uintptr_t)lds + k * 256 + (tg_pos32<B>(i >> 4, k) << 5) + ((i & 15) << 1);
                h[s] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tg_lds_s16x4*>(at));
            }
            const u32x2 lo = __builtin_bit_cast(u32x2, h[0]), hi = __builtin_bit_cast(u32x2, h[1]);
            v[f] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
    } else {
        u32x4 t[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) t[s] = lds_read_b128(lds, (kk * 16 + 4 * lg + s) * 512 + (w * 64 + 4 * li) * 4);
#pragma unroll
        for (int f = 0; f < 4; ++f) v[f] = u32x4{t[0][f], t[1][f], t[2][f], t[3][f]};
    }
}
}   // namespace

// B side index of value j (0..7) of run h (0, 1) of a lane: base(h) + j, held by tile f, accumulator q
template <typename T, bool BMN> struct TgRun {
    static constexpr bool R4 = BMN && sizeof(T) == 4;
    static __device__ __forceinline__ int base(int h, int lg) { return R4 ? 16 * lg + 8 * h : 32 * h + 8 * lg; }
    static constexpr int f(int h, int j) { return R4 ? (j & 3) : 2 * h + (j >> 2); }
    static constexpr int q(int h, int j) { return R4 ? 2 * h + (j >> 2) : (j & 3); }
};

template <typename T, bool AMN, bool BMN, int EPI, bool AL>
__global__ __launch_bounds__(256) void tg_kernel(const TgArgs a, const int tiles_n, const int tiles, const int splits, const long long sps, float* const slab) {
    constexpr int CK = Tr<T>::CK;
    constexpr int BN = EPI == TG_GATED ? 64 : 128;
    constexpr bool PRECISE = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) char smem[2 * TG_TILE];
    char* const la = smem;
    char* const lb = smem + TG_TILE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
    const int li = lane & 15, lg = lane >> 4;
    // blocks: batch-major, then k part, then tile
    const int bs = blockIdx.x / tiles, sp = bs % splits, bt = bs / splits;
    const int t = xcd_remap(blockIdx.x - bs * tiles, tiles);
    const void* const abase = bt == 0 ? a.a.p : a.a.p2;
    const long long m0 = (long long)(t / tiles_n) * 128, n0 = (long long)(t % tiles_n) * BN;

    f32x4 acc[4][4];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int p = 0; p < 4; ++p) acc[f][p] = f32x4{0.f, 0.f, 0.f, 0.f};

    const long long spr = (a.K + CK - 1) / CK;             // steps of one range
    long long step = sp * sps;
    const long long last = step + sps < spr * a.ranges ? step + sps : spr * a.ranges;
    u32x4 ra[4], rb[4];
    auto load = [&]() {
        const bool r1 = step >= spr;
        const long long k0 = (r1 ? step - spr : step) * CK;
        tg_load<T, AMN, false, EPI, AL>(ra, r1 ? a.a.p2 : abase, a.a, m0, a.M, k0, a.K);
        tg_load<T, BMN, true, EPI, AL>(rb, r1 ? a.b.p2 : a.b.p, a.b, n0, a.N, k0, a.K);
    };
    load();
    while (step < last) {
        __syncthreads();                                   // the previous step's fragment reads are done
        tg_store<T, AMN, false>(la, ra);
        tg_store<T, BMN, true>(lb, rb);
        __syncthreads();
        if (++step < last) load();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 fa[4], fb[4];
            tg_frags<T, AMN, false>(fa, la, wm, kk);
            tg_frags<T, BMN, true>(fb, lb, wn, kk);
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int p = 0; p < 4; ++p) mma_b128<T>(acc[f][p], fb[f], fa[p]);
        }
    }

    using Run = TgRun<T, BMN>;
    if constexpr (EPI == TG_STORE || EPI == TG_SLAB) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long n = n0 + wn * 64 + Run::base(h, lg);
            const int nv = a.N - n >= 8 ? 8 : (int)(a.N - n);
            if (nv <= 0) continue;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const long long m = m0 + wm * 64 + ((AMN && sizeof(T) == 4) ? 4 * li + p : 16 * p + li);
                if (m >= a.M) continue;
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = acc[Run::f(h, j)][p][Run::q(h, j)];
                if constexpr (EPI == TG_STORE) tok_stn<T>(reinterpret_cast<T*>(bt == 0 ? a.y : a.y2) + m * a.ldy + n, v, nv);
                else tok_stn<float>(slab + ((long long)(bt * splits + sp) * a.M + m) * a.N + n, v, nv);
            }
        }
    } else if constexpr (EPI == TG_LINEAR) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const TgLinearRow<T> row(a, bt == 0 ? a.y : a.y2, n0 + wn * 64 + Run::base(h, lg));
            if (row.nv <= 0) continue;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const long long m = m0 + wm * 64 + ((AMN && sizeof(T) == 4) ? 4 * li + p : 16 * p + li);
                if (m >= a.M) continue;
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = acc[Run::f(h, j)][p][Run::q(h, j)];
                row(m, v);
            }
        }
    } else {
        // tiles 0, 1 hold 8 gate columns of a lane, tiles 2, 3 the same columns of up
        static_assert(!Run::R4, "gated: k-contiguous weights only");
        const TgGatedRow<T> row(a, n0 + wn * 32 + 8 * lg);
        if (row.nv <= 0) return;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const long long m = m0 + wm * 64 + 16 * p + li;
            if (m >= a.M) continue;
            float g[8], u[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                g[j] = acc[j >> 2][p][j & 3];
                u[j] = acc[2 + (j >> 2)][p][j & 3];
            }
            row(m, g, u);
        }
    }
}

// y = sum of a product's k parts in their order, rounded; batch 1 goes to y2
template <typename T> __global__ __launch_bounds__(256) void tg_slab_kernel(const TgArgs a, const float* __restrict__ slab, int splits) {
    const long long per = (a.N + 7) >> 3;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.M * per * a.batches) return;
    const long long row = id / per, n = (id - row * per) * 8;
    const int nv = a.N - n >= 8 ? 8 : (int)(a.N - n);
    const int bt = row >= a.M ? 1 : 0;
    const long long m = row - bt * a.M;
    const float* p = slab + ((long long)bt * splits * a.M + m) * a.N + n;
    float v[8];
    tok_ldn<float>(p, v, nv);
    for (int s = 1; s < splits; ++s) {
        float t[8];
        tok_ldn<float>(p + (long long)s * a.M * a.N, t, nv);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += t[j];
    }
    tok_stn<T>(reinterpret_cast<T*>(bt == 0 ? a.y : a.y2) + m * a.ldy + n, v, nv);
}

int tg_slab_sum(int dtype, const TgArgs& a, const float* slab, int splits, hipStream_t stream) {
    const long long n = (a.M * ((a.N + 7) / 8) * a.batches + 255) / 256;
    MIS_REQUIRE(n < (1ll << 31), MIS_EUNSUPPORTED, "token product: the grid is too large");
    if (dtype == MIS_BF16) hipLaunchKernelGGL(tg_slab_kernel<__bf16>, dim3((unsigned)n), dim3(256), 0, stream, a, slab, splits);
    else hipLaunchKernelGGL(tg_slab_kernel<float>, dim3((unsigned)n), dim3(256), 0, stream, a, slab, splits);
    MIS_LAUNCH_CHECK("token product (sum of k parts)");
    return MIS_OK;
}

namespace {
// How a product is cut.  Costs in microseconds of one CU: a 256 x 256 step of 64 k takes ~1 us, four 128 x 128 steps as much (bf16; f32 16 times that); a k part costs its slab's write and
// read at the copy rate; a tile's epilogue about 3 steps.
struct TgCut {
    bool pp;
    int splits;
    double us;
};
TgCut tg_cut_one(int dtype, bool pp, bool may_split, long long M, long long N, long long K, int ranges, int batches, int cols) {
    const int T = pp ? 256 : 128;
    const long long items = ((M + T - 1) / T) * ((N + cols - 1) / cols) * batches, steps = ((K + 63) / 64) * ranges;
    const double step = (pp ? 1.0 : 0.45) * (dtype == MIS_BF16 ? 1.0 : 14.0), slots = pp ? 256.0 : 512.0;
    TgCut best{pp, 1, 1e30};
    if (const int forced = mis_sw(SW_TOK_SPLITS); may_split && forced > 0) return TgCut{pp, (int)(forced < steps ? forced : steps), 0.0};
    for (int s = 1; s <= (may_split ? 32 : 1) && (s == 1 || steps / s >= 4); ++s) {
        const double rounds = (double)((items * s + (long long)slots - 1) / (long long)slots);
        double us = rounds * ((double)((steps + s - 1) / s) * step + 3.0 * (pp ? 1.0 : 0.5));
        if (s > 1) us += 3.0 + 8.0 * s * (double)M * (double)N * batches / 4.7e6;
        if (us < best.us * 0.97) best = TgCut{pp, s, us};
    }
    return best;
}
TgCut tg_cut(int dtype, bool aligned, bool may_split, long long M, long long N, long long K, int ranges, int batches, bool gated) {
    const TgCut g = tg_cut_one(dtype, false, may_split, M, N, K, ranges, batches, gated ? 64 : 128);
    const int forced = mis_sw(SW_TOK_TILE);
    if (dtype != MIS_BF16 || !aligned || forced == 1) return g;
    const TgCut p = tg_cut_one(dtype, true, may_split, M, N, K, ranges, batches, gated ? 128 : 256);
    return p.us <= g.us || forced == 2 ? p : g;
}
// 16-byte chunks from 16-byte addresses, 32-bit offsets inside a tile; a k-contiguous operand's k, the other kind's own index must be whole chunks
bool tg_pp_ok(const TgArgs& a, int a_mn, int b_mn) {
    auto ok = [&](const TgOperand& o, int mn, long long I) {
        return ((uintptr_t)o.p | (uintptr_t)o.p2 | (size_t)(o.ld * 2)) % 16 == 0 && o.ld <= (1 << 21) && (mn ? I : a.K) % 8 == 0;
    };
    return ok(a.a, a_mn, a.M) && ok(a.b, b_mn, a.N);
}

template <typename T, bool AMN, bool BMN, int EPI> int tg_go(const TgArgs& a, int splits, float* slab, hipStream_t stream) {
    constexpr int BN = EPI == TG_GATED ? 64 : 128;
    const long long tm = (a.M + 127) / 128, tn = (a.N + BN - 1) / BN, steps = (a.K + Tr<T>::CK - 1) / Tr<T>::CK * a.ranges;
    const long long sps = (steps + splits - 1) / splits;
    splits = (int)((steps + sps - 1) / sps);                       // (no part is empty)
    MIS_REQUIRE(tm < (1ll << 31) && tn < (1ll << 31) && tm * tn * a.batches < (1ll << 31) / splits, MIS_EUNSUPPORTED, "token product: %lld x %lld tiles are more than a grid holds", tm, tn);
    auto al = [](const TgOperand& o) { return ((uintptr_t)o.p | (uintptr_t)o.p2 | (size_t)(o.ld * (long long)sizeof(T))) % 16 == 0; };
    const dim3 grid((unsigned)(tm * tn * a.batches * splits));
    if (al(a.a) && al(a.b))
        hipLaunchKernelGGL((tg_kernel<T, AMN, BMN, EPI, true>), grid, dim3(256), 0, stream, a, (int)tn, (int)(tm * tn), splits, sps, slab);
    else
        hipLaunchKernelGGL((tg_kernel<T, AMN, BMN, EPI, false>), grid, dim3(256), 0, stream, a, (int)tn, (int)(tm * tn), splits, sps, slab);
    MIS_LAUNCH_CHECK("token product");
    if constexpr (EPI == TG_SLAB) return tg_slab_sum(sizeof(T) == 2 ? MIS_BF16 : MIS_F32, a, slab, splits, stream);
    return MIS_OK;
}
template <typename T> int tg_pick(int a_mn, int b_mn, int epi, const TgArgs& a, int splits, float* slab, hipStream_t stream) {
    if (epi == TG_GATED) return tg_go<T, false, false, TG_GATED>(a, 1, nullptr, stream);
    if (epi == TG_LINEAR) return tg_go<T, false, false, TG_LINEAR>(a, 1, nullptr, stream);
    if (splits == 1) return a_mn ? tg_go<T, true, true, TG_STORE>(a, 1, nullptr, stream) : tg_go<T, false, true, TG_STORE>(a, 1, nullptr, stream);
    return a_mn ? tg_go<T, true, true, TG_SLAB>(a, splits, slab, stream) : tg_go<T, false, true, TG_SLAB>(a, splits, slab, stream);
}
}   // namespace

size_t tg_slab_bytes(int dtype, long long M, long long N, long long K, int ranges, int batches) {
    size_t most = 0;
    for (int al = 0; al < 2; ++al) {
        const TgCut c = tg_cut(dtype, al == 1, true, M, N, K, ranges, batches, false);
        const size_t n = c.splits > 1 ? tok_align((size_t)c.splits * batches * M * N * 4) : 0;
        if (n > most) most = n;
    }
    return most;
}

int tg_launch(int dtype, int a_mn, int b_mn, int epi, const TgArgs& a, float* slab, hipStream_t stream) {
    const TgCut c = tg_cut(dtype, tg_pp_ok(a, a_mn, b_mn), epi == TG_STORE, a.M, a.N, a.K, a.ranges, a.batches, epi == TG_GATED);
    if (c.pp) return tg_pp_launch(a_mn, b_mn, epi, a, slab, c.splits, stream);
    return dtype == MIS_BF16 ? tg_pick<__bf16>(a_mn, b_mn, epi, a, c.splits, slab, stream) : tg_pick<float>(a_mn, b_mn, epi, a, c.splits, slab, stream);
}
