// Forward token products with few rows (serving: one token, or a handful of sequences' next tokens): y = act(x W^T + b) + res and h = act(g) u for M <= 32.
//
// The weights are read once and are all there is to read, so the kernel is a stream of them: a block owns 16 columns (gated: the same 16 of gate and of up; 32 for more than 16 rows), its
// waves take turns along k in units of 128 bytes per row, and a weight fragment goes from global memory straight into the MFMA's row side - no LDS, no barrier - against the rows of x,
// which come out of the L2.  The waves' partial sums meet in LDS in wave order, then the epilogue runs on runs of 8 columns.  As many waves per block as bring ~2000 of them onto the
// chip, at most 8 where a lane holds two tiles of rows (16 leave it 128 registers, and its fragments spill).
//
// Bound by the weights: one row of 8192 x 8192 bf16 (134 MB) 30 us, 4.5 TB/s; f32 57 us, 4.7 TB/s.  Up to which rows, against 64 x 64 tiles with k parts (tok_gemm.hip), us here / there:
//      rows   bf16 2048 -> 8192   gated 2048 -> 2 x 8192   8192 -> 8192   f32 1024 -> 4096   2048 -> 8192   8192 -> 8192
//        1          8.1 / 13.1          13.7 / 17.5          30 / 26         8.3 / 13.2        15 / 25        57 / 74
//       16          9.9 / 13.1          15.2 / 17.1          35 / 27         8.2 / 13.2        18 / 25        70 / 75
//       32         10.7 / 13.1          21.3 / 17.6          38 / 28        12.3 / 13.3        24 / 26        73 / 75
//       48         14.2 / 13.1          23.3 / 17.8          43 / 28        18.7 / 13.3        38 / 27       134 / 77        (with four tiles of rows per lane)
// - two launches and a sum where this is one.  The limit is one number of rows whatever the weights are: it loses 4 to 10 us on the largest bf16 ones and at 32 gated rows, and wins 1 to 17
// on smaller ones and in f32.
#include "tok_epilogue.hpp"
#include "tok_product_plan.hpp"

namespace {
template <typename T, bool AL> __device__ __forceinline__ u32x4 sk_chunk(const T* p, long long n) {
    constexpr int EPC = Tr<T>::EPC;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n >= EPC) {
        if constexpr (AL) v = *reinterpret_cast<const u32x4*>(p);
        else v = tok_ld16<T>(p);
    } else if (!AL && n > 0) {          // (AL: k is a multiple of a chunk)
        float f[EPC];
#pragma unroll
        for (int i = 0; i < EPC; ++i) f[i] = i < n ? ld_elem<T>(p + i) : 0.f;
        v = pack_chunk<T>(f);
    }
    return v;
}
}   // namespace

// NT tiles of 16 columns (gated: gate, up), MT tiles of 16 rows, blockDim.x / 64 waves along k
template <typename T, int NT, int MT, bool GATED, bool AL>
__global__ __launch_bounds__(MT == 1 ? 1024 : 512) void tok_skinny_kernel(const TgArgs a) {
    constexpr int EPC = Tr<T>::EPC, S = 4 * EPC;          // k of one MFMA step: 64 bytes per row
    extern __shared__ __attribute__((aligned(16))) float part[];          // [wave][NT][MT][16 m][16 n]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), W = blockDim.x >> 6;
    const int li = lane & 15, lg = lane >> 4;
    const long long n0 = (long long)blockIdx.x * (GATED ? 16 : 16 * NT);

    // rows past the end read the last one (their results are not stored)
    const T* wp[NT];
    const T* xp[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const long long n = GATED ? n0 + li : n0 + 16 * t + li;
        wp[t] = reinterpret_cast<const T*>(GATED && t == 1 ? a.b.p2 : a.b.p) + (n < a.N ? n : a.N - 1) * a.b.ld + lg * EPC;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const long long r = 16 * m + li;
        xp[m] = reinterpret_cast<const T*>(a.a.p) + (r < a.M ? r : a.M - 1) * a.a.ld + lg * EPC;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};

    const long long units = (a.K + 2 * S - 1) / (2 * S);
    u32x4 fw[NT][2], fx[MT][2];
    auto load = [&](u32x4 (&w)[NT][2], u32x4 (&x)[MT][2], long long u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long k = (2 * u + h) * S, left = a.K - k - lg * EPC;
#pragma unroll
            for (int t = 0; t < NT; ++t) w[t][h] = sk_chunk<T, AL>(wp[t] + k, left);
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m][h] = sk_chunk<T, AL>(xp[m] + k, left);
        }
    };
    auto mma = [&](const u32x4 (&w)[NT][2], const u32x4 (&x)[MT][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int m = 0; m < MT; ++m) mma_b128<T>(acc[t][m], w[t][h], x[m][h]);
    };
    long long u = wave;
    if (u < units) load(fw, fx, u);
    while (u < units) {
        u32x4 gw[NT][2], gx[MT][2];
        const long long v = u + W;
        if (v < units) load(gw, gx, v);
        mma(fw, fx);
        if (v >= units) break;
        u = v + W;
        if (u < units) load(fw, fx, u);
        mma(gw, gx);
    }

#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) *reinterpret_cast<f32x4*>(part + (((wave * NT + t) * MT + m) * 16 + li) * 16 + 4 * lg) = acc[t][m];
    __syncthreads();
    auto sum8 = [&](int t, int row, int half, float (&v)[8]) {
        const float* p = part + ((t * MT + (row >> 4)) * 16 + (row & 15)) * 16 + 8 * half;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        for (int w = 0; w < W; ++w, p += NT * MT * 256)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += p[j];
    };
    const int rows = a.M < 16 * MT ? (int)a.M : 16 * MT;
    if constexpr (GATED) {
        for (int id = threadIdx.x; id < rows * 2; id += blockDim.x) {
            const TgGatedRow<T> row(a, n0 + 8 * (id & 1));
            if (row.nv <= 0) continue;
            float g[8], q[8];
            sum8(0, id >> 1, id & 1, g);
            sum8(1, id >> 1, id & 1, q);
            row(id >> 1, g, q);
        }
    } else {
        for (int id = threadIdx.x; id < rows * 2 * NT; id += blockDim.x) {
            const int h = id % (2 * NT), r = id / (2 * NT);
            const TgLinearRow<T> row(a, a.y, n0 + 8 * h, true);
            if (row.nv <= 0) continue;
            float v[8];
            sum8(h >> 1, r, h & 1, v);
            row(r, v);
        }
    }
}

namespace {
template <typename T, int NT, int MT, bool GATED, bool AL> int sk_go(const TgArgs& a, hipStream_t stream) {
    const long long cols = GATED ? 16 : 16 * NT, blocks = (a.N + cols - 1) / cols, units = (a.K + 8 * Tr<T>::EPC - 1) / (8 * Tr<T>::EPC);
    int W = 1;          // (at most 2^25 blocks: tg_few_rows)
    while (W < (MT == 1 ? 16 : 8) && blocks * W < 2048 && 2 * W <= units) W *= 2;
    hipLaunchKernelGGL((tok_skinny_kernel<T, NT, MT, GATED, AL>), dim3((unsigned)blocks), dim3(64 * W), (size_t)W * NT * MT * 1024, stream, a);
    MIS_LAUNCH_CHECK("token product (few rows)");
    return MIS_OK;
}
template <typename T, bool GATED, bool AL> int sk_rows(const TgArgs& a, hipStream_t stream) {
    if (a.M <= 16) return sk_go<T, GATED ? 2 : 1, 1, GATED, AL>(a, stream);
    return sk_go<T, 2, 2, GATED, AL>(a, stream);
}
template <typename T> int sk_type(int epi, const TgArgs& a, bool al, hipStream_t stream) {
    if (epi == TG_GATED) return al ? sk_rows<T, true, true>(a, stream) : sk_rows<T, true, false>(a, stream);
    return al ? sk_rows<T, false, true>(a, stream) : sk_rows<T, false, false>(a, stream);
}
}   // namespace

int tok_product_skinny(int dtype, int epi, const TgArgs& a, bool aligned, hipStream_t stream) {
    return dtype == MIS_BF16 ? sk_type<__bf16>(epi, a, aligned, stream) : sk_type<float>(epi, a, aligned, stream);
}
