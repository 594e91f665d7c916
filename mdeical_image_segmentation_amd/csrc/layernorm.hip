// Layer norm over the channels of a token, forward and backward (include/misamd.h: mis_layernorm_*).
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) rstd, y = xh gamma + beta
//   dx = rstd (t - mean(t) - xh mean(t xh)), t = dy gamma;   dgamma = sum_rows dy xh, dbeta = sum_rows dy
// All statistics and sums are f32; the variance is that of the centred values (no E[x^2] - mu^2 cancellation).
//
// About ten operations a value: bandwidth bounds both directions, so a row is read once and lives in registers (runs of 8 values per lane) between the passes over it.  A row belongs to as
// few lanes as hold it: 8 to 64 lanes of a wave up to 2048 values (no barrier at all), the four waves of a block up to 8192; wider ones are read again for each pass and stay in the caches.
// Backward: one kernel reads x and dy once, writes dx and keeps these lanes' part of dgamma and dbeta in registers over all its rows; the blocks' partial rows are then added in a
// fixed order.  Rows x width, us forward / backward and the rates of x + y, x + dy + dx (a large copy: 4.7 TB/s):
//                       bf16                                     f32
//      65536 x 96        9.0 / 15.1   2.8, 2.5 TB/s             10.5 / 18.2   4.8, 4.1 TB/s      (64 lanes a row: 22.8 / 34.4, 23.6 / 29.8)
//      32768 x 1024     24.3 / 41.6   5.5, 4.8                  42.9 / 77.7   6.3, 5.2
//      16384 x 2048     26.4 / 45.0   5.1, 4.5                  44.2 / 85.4   6.1, 4.7           (four waves a row: 29.2 / 57.8, 40.3 / 77.7)
//      8192 x 4096      23.7 / 44.5   5.7, 4.5                  43.4 / 82.2   6.2, 4.9           (read again: 28.6 / 72.1, 59.6 / 141)
//      2048 x 16384     39.7 / 80.4   3.4, 2.5                  75.9 / 141    3.5, 2.9
//      8192 x 2056      19.2 / 34.3   3.5, 2.9                  24.0 / 41.7   5.6, 4.9           (just past a power of two: half of the lanes have nothing)
#include <type_traits>

#include "tok_common.hpp"

namespace {
constexpr int LN_THREADS = 256;

// sum over the block's 256 threads, the same order whatever the wave timing; `red` is reusable after the call
__device__ __forceinline__ float ln_block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
}   // namespace

namespace {
// sum over the L lanes that share a row (256: the block; `red` is then reusable behind the next barrier)
template <int L> __device__ __forceinline__ float ln_row_sum(float v, float* red) {
    if constexpr (L < 64) {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    } else {
        v = wave_sum(v);
    }
    if constexpr (L == 256) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (red[0] + red[1]) + (red[2] + red[3]);
    }
    return v;
}
}   // namespace

// L lanes per row (8, 16, 32, 64: 256 / L rows a block; 256: one), NV runs of 8 values per lane: D <= 8 L NV
template <typename T, int L, int NV>
__global__ __launch_bounds__(LN_THREADS) void ln_fwd_row_kernel(const T* __restrict__ x, long long ldx, long long M, int D, float eps, const float* __restrict__ gamma,
                                                                const float* __restrict__ beta, T* __restrict__ y, long long ldy, float* __restrict__ mean,
                                                                float* __restrict__ rstd) {
    __shared__ float red[2][4];
    const int lane = threadIdx.x & (L - 1);
    const long long r = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (r >= M) return;                                      // (a row's lanes go together)
    float f[NV][8];
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * L + lane) * 8;
        tok_ldn<T>(x + r * ldx + c, f[v], D - c);            // (0 past the row's end)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += f[v][i];
    }
    const float mu = ln_row_sum<L>(s, red[0]) / D;
    s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f[v][i] = (v * L + lane) * 8 + i < D ? f[v][i] - mu : 0.f;
            s += f[v][i] * f[v][i];
        }
    const float rs = 1.f / sqrtf(ln_row_sum<L>(s, red[1]) / D + eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * L + lane) * 8;
        if (c < D) {
            float g[8], b[8];
            if (gamma != nullptr) tok_ldn<float>(gamma + c, g, D - c);
            if (beta != nullptr) tok_ldn<float>(beta + c, b, D - c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[v][i] *= rs;
                if (gamma != nullptr) f[v][i] *= g[i];
                if (beta != nullptr) f[v][i] += b[i];
            }
            tok_stn<T>(y + r * ldy + c, f[v], D - c);
        }
    }
    if (lane == 0) {
        if (mean != nullptr) mean[r] = mu;
        if (rstd != nullptr) rstd[r] = rs;
    }
}

template <typename T, int L, int NV>
__global__ __launch_bounds__(LN_THREADS) void ln_bwd_row_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x, long long ldx, long long M, int D,
                                                                const float* __restrict__ gamma, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                T* __restrict__ dx, long long lddx, float* __restrict__ pg, float* __restrict__ pb) {
    __shared__ float red[2][2][4];
    __shared__ float acc[L == 256 ? 1 : LN_THREADS * 8];
    const int lane = threadIdx.x & (L - 1), sub = threadIdx.x / L;
    constexpr int per = 256 / L;
    float g[NV][8], sg[NV][8], sb[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * L + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[v][i] = 1.f, sg[v][i] = sb[v][i] = 0.f;
        if (gamma != nullptr && c < D) tok_ldn<float>(gamma + c, g[v], D - c);
    }
    int flip = 0;
    for (long long r = (long long)blockIdx.x * per + sub; r < M; r += (long long)gridDim.x * per) {          // (a row's lanes go together)
        const float mu = mean[r], rs = rstd[r];
        float f[NV][8], d[NV][8];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * L + lane) * 8;
            tok_ldn<T>(x + r * ldx + c, f[v], D - c);
            tok_ldn<T>(dy + r * lddy + c, d[v], D - c);      // (0 past the row's end: nothing is added there)
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float xh = (f[v][i] - mu) * rs, e = d[v][i];
                sg[v][i] += e * xh;
                sb[v][i] += e;
                f[v][i] = xh;
                d[v][i] = e * g[v][i];
                s1 += d[v][i];
                s2 += d[v][i] * xh;
            }
        if (dx != nullptr) {
            const float m1 = ln_row_sum<L>(s1, red[flip][0]) / D, m2 = ln_row_sum<L>(s2, red[flip][1]) / D;
            flip ^= 1;                                       // (the next round's sums go elsewhere: two barriers lie between two uses)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * L + lane) * 8;
                if (c < D) {
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = rs * (d[v][i] - m1 - f[v][i] * m2);
                    tok_stn<T>(dx + r * lddx + c, o, D - c);
                }
            }
        }
    }
    // this block's partial rows; those of its 256 / L rows are added in their order
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* const out = which == 0 ? pg : pb;
        if (out == nullptr) continue;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * L + lane) * 8;
            if constexpr (L < 256) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[(sub * 8 + i) * L + lane] = which == 0 ? sg[v][i] : sb[v][i];
                __syncthreads();
                for (int q = threadIdx.x; q < 8 * L; q += LN_THREADS) {
                    const int col = (v * L + q % L) * 8 + q / L;
                    float t = acc[q];
#pragma unroll
                    for (int k = 1; k < per; ++k) t += acc[k * 8 * L + q];
                    if (col < D) out[(long long)blockIdx.x * D + col] = t;
                }
            } else if (c < D) {
                tok_stn<float>(out + (long long)blockIdx.x * D + c, which == 0 ? sg[v] : sb[v], D - c);
            }
        }
    }
}

// Any width: a block per row, the row read again for each pass (it stays in the caches)
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_fwd_kernel(const T* __restrict__ x, long long ldx, int D, float eps, const float* __restrict__ gamma,
                                                            const float* __restrict__ beta, T* __restrict__ y, long long ldy, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float red[4];
    const long long r = blockIdx.x;
    const T* xr = x + r * ldx;
    T* yr = y + r * ldy;
    float s = 0.f;
    for (int c = threadIdx.x * 8; c < D; c += LN_THREADS * 8) {
        float f[8];
        tok_ldn<T>(xr + c, f, D - c);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += f[i];
    }
    const float mu = ln_block_sum(s, red) / D;
    s = 0.f;
    for (int c = threadIdx.x * 8; c < D; c += LN_THREADS * 8) {
        float f[8];
        tok_ldn<T>(xr + c, f, D - c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = f[i] - mu;
            if (c + i < D) s += e * e;
        }
    }
    const float rs = 1.f / sqrtf(ln_block_sum(s, red) / D + eps);
    for (int c = threadIdx.x * 8; c < D; c += LN_THREADS * 8) {
        float f[8], g[8], b[8];
        tok_ldn<T>(xr + c, f, D - c);
        if (gamma != nullptr) tok_ldn<float>(gamma + c, g, D - c);
        if (beta != nullptr) tok_ldn<float>(beta + c, b, D - c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f[i] = (f[i] - mu) * rs;
            if (gamma != nullptr) f[i] *= g[i];
            if (beta != nullptr) f[i] += b[i];
        }
        tok_stn<T>(yr + c, f, D - c);
    }
    if (threadIdx.x == 0) {
        if (mean != nullptr) mean[r] = mu;
        if (rstd != nullptr) rstd[r] = rs;
    }
}

template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_bwd_dx_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x, long long ldx, int D, const float* __restrict__ gamma,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, long long lddx) {
    __shared__ float red[4];
    const long long r = blockIdx.x;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
        float m1 = 0.f, m2 = 0.f;
        if (pass == 1) {
            m1 = ln_block_sum(s1, red) / D;
            m2 = ln_block_sum(s2, red) / D;
        }
        for (int c = threadIdx.x * 8; c < D; c += LN_THREADS * 8) {
            float f[8], d[8], g[8];
            tok_ldn<T>(x + r * ldx + c, f, D - c);
            tok_ldn<T>(dy + r * lddy + c, d, D - c);
            if (gamma != nullptr) tok_ldn<float>(gamma + c, g, D - c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float xh = (f[i] - mu) * rs, t = gamma != nullptr ? d[i] * g[i] : d[i];
                if (pass == 0) {
                    if (c + i < D) {
                        s1 += t;
                        s2 += t * xh;
                    }
                } else {
                    f[i] = rs * (t - m1 - xh * m2);
                }
            }
            if (pass == 1) tok_stn<T>(dx + r * lddx + c, f, D - c);
        }
    }
}

// partial sums of dgamma / dbeta: a block owns 64 columns and `rows` rows
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_bwd_param_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x, long long ldx, long long M, int D,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ pg, float* __restrict__ pb,
                                                                  long long rows, int nrb) {
    __shared__ float red[2][32][64];
    const int cg = threadIdx.x & 7, rl = threadIdx.x >> 3;
    const long long rb = blockIdx.x % nrb;
    const int c = (int)(blockIdx.x / nrb) * 64 + cg * 8;
    float sg[8], sb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sg[i] = sb[i] = 0.f;
    const long long m1 = (rb + 1) * rows < M ? (rb + 1) * rows : M;
    if (c < D)
        for (long long m = rb * rows + rl; m < m1; m += 32) {
            float f[8], d[8];
            const float mu = mean[m], rs = rstd[m];
            tok_ldn<T>(x + m * ldx + c, f, D - c);
            tok_ldn<T>(dy + m * lddy + c, d, D - c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sg[i] += d[i] * ((f[i] - mu) * rs);
                sb[i] += d[i];
            }
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        red[0][rl][cg * 8 + i] = sg[i];
        red[1][rl][cg * 8 + i] = sb[i];
    }
    __syncthreads();
    const int which = threadIdx.x >> 6, cc = threadIdx.x & 63;
    const int col = (int)(blockIdx.x / nrb) * 64 + cc;
    if (which < 2 && col < D) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) s += red[which][r][cc];
        float* const out = which == 0 ? pg : pb;
        if (out != nullptr) out[rb * D + col] = s;
    }
}

namespace {
// a grid holds fewer than 2^32 work-items: kernels that give every row its lanes are launched again behind this many
constexpr long long LN_ITEMS = 1ll << 31;
inline long long ln_rows(long long M, int D) {
    long long r = 64;
    while ((M + r - 1) / r > 512 || (M + r - 1) / r * ((D + 63) / 64) * LN_THREADS > LN_ITEMS) r *= 2;
    return r;
}
// lanes per row and runs per lane that a width takes; 0: the kernels for any width
inline int ln_lanes(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : (D <= 256 ? 32 : (D <= 2048 ? 64 : (D <= 8192 ? 256 : 0)))); }
inline int ln_runs(int D) { return (D + 8 * ln_lanes(D) - 1) / (8 * ln_lanes(D)); }
// Blocks of the backward pass = partial rows of the parameter gradients: 1024 where the registers let four blocks onto a CU and 16-byte loads (bf16: a lane has half of f32's bytes in
// flight) need them, else 512.  512 / 1024 / 2048 blocks, us: bf16 8192 x 2056 49 / 34 / 43, 32768 x 1024 46 / 42 / 49, 16384 x 2048 45 / 53 / 53; f32 32768 x 1024 78 / 82 / 87,
// 4096 x 8192 91 / 99 / 99
constexpr int LN_PART = 512, LN_PART_LIGHT = 1024;
inline long long ln_parts(int dtype, long long M, int D) {
    const int n = ln_lanes(D);
    if (n == 0) return (M + ln_rows(M, D) - 1) / ln_rows(M, D);
    const long long blocks = (M * n + 255) / 256, most = D <= 256 || (dtype == MIS_BF16 && ln_runs(D) <= 2) ? LN_PART_LIGHT : LN_PART;
    return blocks < most ? blocks : most;
}
template <int V> using ln_int = std::integral_constant<int, V>;
template <typename T, typename F> int ln_by_width(int D, F&& f) {
    const int w = ln_lanes(D), n = ln_runs(D);
    if (w == 8) return f(ln_int<8>{}, ln_int<1>{});
    if (w == 16) return f(ln_int<16>{}, ln_int<1>{});
    if (w == 32) return f(ln_int<32>{}, ln_int<1>{});
    if (w == 64) return n == 1 ? f(ln_int<64>{}, ln_int<1>{}) : n == 2 ? f(ln_int<64>{}, ln_int<2>{}) : n == 3 ? f(ln_int<64>{}, ln_int<3>{}) : f(ln_int<64>{}, ln_int<4>{});
    return n == 2 ? f(ln_int<256>{}, ln_int<2>{}) : n == 3 ? f(ln_int<256>{}, ln_int<3>{}) : f(ln_int<256>{}, ln_int<4>{});          // (one run of a block: up to 2048, which a wave takes)
}
// f(first row, rows) for as many rows at a time as one grid of L lanes a row holds
template <int L, typename F> int ln_by_rows(long long M, F&& f) {
    for (long long r = 0; r < M; r += LN_ITEMS / L)
        if (const int rc = f(r, M - r < LN_ITEMS / L ? M - r : LN_ITEMS / L)) return rc;
    return MIS_OK;
}
template <typename T>
int ln_fwd(const void* x_, long long ldx, long long M, int D, float eps, const float* gamma, const float* beta, void* y_, long long ldy, float* mean, float* rstd, hipStream_t stream) {
    const T* const x = (const T*)x_;
    T* const y = (T*)y_;
    auto at = [](float* p, long long r) { return p != nullptr ? p + r : nullptr; };
    if (ln_lanes(D) == 0)
        return ln_by_rows<LN_THREADS>(M, [&](long long r, long long rows) {
            hipLaunchKernelGGL((ln_fwd_kernel<T>), dim3((unsigned)rows), dim3(LN_THREADS), 0, stream, x + r * ldx, ldx, D, eps, gamma, beta, y + r * ldy, ldy, at(mean, r), at(rstd, r));
            MIS_LAUNCH_CHECK("mis_layernorm_fwd");
            return (int)MIS_OK;
        });
    return ln_by_width<T>(D, [&](auto w, auto n) {
        constexpr int L = decltype(w)::value, NV = decltype(n)::value;
        return ln_by_rows<L>(M, [&](long long r, long long rows) {
            hipLaunchKernelGGL((ln_fwd_row_kernel<T, L, NV>), dim3((unsigned)((rows * L + 255) / 256)), dim3(LN_THREADS), 0, stream, x + r * ldx, ldx, rows, D, eps, gamma, beta, y + r * ldy, ldy,
                               at(mean, r), at(rstd, r));
            MIS_LAUNCH_CHECK("mis_layernorm_fwd");
            return (int)MIS_OK;
        });
    });
}
template <typename T>
int ln_bwd(const void* dy_, long long lddy, const void* x_, long long ldx, long long M, int D, const float* gamma, const float* mean, const float* rstd, void* dx_, long long lddx, float* pg,
           float* pb, hipStream_t stream) {
    const T *const dy = (const T*)dy_, *const x = (const T*)x_;
    T* const dx = (T*)dx_;
    const long long parts = ln_parts(sizeof(T) == 2 ? MIS_BF16 : MIS_F32, M, D);
    if (ln_lanes(D) == 0) {
        if (dx != nullptr)
            if (const int rc = ln_by_rows<LN_THREADS>(M, [&](long long r, long long rows) {
                    hipLaunchKernelGGL((ln_bwd_dx_kernel<T>), dim3((unsigned)rows), dim3(LN_THREADS), 0, stream, dy + r * lddy, lddy, x + r * ldx, ldx, D, gamma, mean + r, rstd + r,
                                       dx + r * lddx, lddx);
                    MIS_LAUNCH_CHECK("mis_layernorm_bwd");
                    return (int)MIS_OK;
                }))
                return rc;
        if (pg != nullptr || pb != nullptr)
            hipLaunchKernelGGL((ln_bwd_param_kernel<T>), dim3((unsigned)(parts * ((D + 63) / 64))), dim3(LN_THREADS), 0, stream, dy, lddy, x, ldx, M, D, mean, rstd, pg, pb, ln_rows(M, D),
                               (int)parts);
        MIS_LAUNCH_CHECK("mis_layernorm_bwd");
        return MIS_OK;
    }
    return ln_by_width<T>(D, [&](auto w, auto n) {
        constexpr int L = decltype(w)::value, NV = decltype(n)::value;
        hipLaunchKernelGGL((ln_bwd_row_kernel<T, L, NV>), dim3((unsigned)parts), dim3(LN_THREADS), 0, stream, dy, lddy, x, ldx, M, D, gamma, mean, rstd, dx, lddx, pg, pb);
        MIS_LAUNCH_CHECK("mis_layernorm_bwd");
        return (int)MIS_OK;
    });
}
int ln_check(const char* who, int dtype, long long M, int D) {
    MIS_REQUIRE(dtype == MIS_F32 || dtype == MIS_BF16, MIS_EINVAL, "%s: dtype must be MIS_F32 or MIS_BF16", who);
    MIS_REQUIRE(M >= 0 && D >= 1, MIS_EINVAL, "%s: needs rows >= 0 and a width >= 1 (got %lld, %d)", who, M, D);
    MIS_REQUIRE(M < (1ll << 31), MIS_EUNSUPPORTED, "%s: %lld rows are more than its grids hold", who, M);
    MIS_REQUIRE(D <= (1 << 22), MIS_EUNSUPPORTED, "%s: width %d is over 2^22", who, D);
    return MIS_OK;
}
}   // namespace

extern "C" int mis_layernorm_fwd(int dtype, const void* x, long long ldx, long long M, int D, float eps, const float* gamma, const float* beta, void* y, long long ldy,
                                 float* mean, float* rstd, void* stream) {
    if (const int rc = ln_check("mis_layernorm_fwd", dtype, M, D)) return rc;
    if (M == 0) return MIS_OK;
    MIS_REQUIRE(x != nullptr && y != nullptr, MIS_EINVAL, "mis_layernorm_fwd: null pointer");
    MIS_REQUIRE(ldx >= D && ldy >= D, MIS_EINVAL, "mis_layernorm_fwd: a row stride is below the width");
    const hipStream_t s = (hipStream_t)stream;
    return dtype == MIS_BF16 ? ln_fwd<__bf16>(x, ldx, M, D, eps, gamma, beta, y, ldy, mean, rstd, s) : ln_fwd<float>(x, ldx, M, D, eps, gamma, beta, y, ldy, mean, rstd, s);
}

extern "C" size_t mis_layernorm_bwd_workspace_bytes(int dtype, long long M, int D) {
    if (ln_check("mis_layernorm_bwd", dtype, M, D) != MIS_OK || M == 0) return 0;
    return 2 * tok_align((size_t)ln_parts(dtype, M, D) * D * 4);
}

extern "C" int mis_layernorm_bwd(int dtype, const void* dy, long long lddy, const void* x, long long ldx, long long M, int D, const float* gamma, const float* mean,
                                 const float* rstd, void* dx, long long lddx, float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes, void* stream_) {
    const hipStream_t stream = (hipStream_t)stream_;
    if (const int rc = ln_check("mis_layernorm_bwd", dtype, M, D)) return rc;
    MIS_REQUIRE(M == 0 || (dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr), MIS_EINVAL, "mis_layernorm_bwd: null pointer");
    MIS_REQUIRE(lddy >= D && ldx >= D && (dx == nullptr || lddx >= D), MIS_EINVAL, "mis_layernorm_bwd: a row stride is below the width");
    const long long parts = M > 0 ? ln_parts(dtype, M, D) : 0;
    const bool params = dgamma != nullptr || dbeta != nullptr;
    const size_t half = tok_align((size_t)parts * D * 4);
    MIS_REQUIRE(!params || M == 0 || (workspace != nullptr && workspace_bytes >= 2 * half), MIS_EINVAL, "mis_layernorm_bwd: the workspace has %zu bytes, %zu are needed",
                workspace_bytes, 2 * half);
    float* const pg = dgamma != nullptr ? (float*)workspace : nullptr;
    float* const pb = dbeta != nullptr ? (float*)((char*)workspace + half) : nullptr;
    if (M > 0 && (params || dx != nullptr)) {
        const int rc = dtype == MIS_BF16 ? ln_bwd<__bf16>(dy, lddy, x, ldx, M, D, gamma, mean, rstd, dx, lddx, pg, pb, stream)
                                         : ln_bwd<float>(dy, lddy, x, ldx, M, D, gamma, mean, rstd, dx, lddx, pg, pb, stream);
        if (rc != MIS_OK) return rc;
    }
    // (no rows: the sums are over nothing and the gradients zero)
    if (params) return tok_column_sums(pg, pb, parts, D, dgamma, dbeta, stream);
    return MIS_OK;
}
