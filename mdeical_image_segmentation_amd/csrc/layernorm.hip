// Layer norm over the channels of a token, forward and backward (include/misamd.h: mis_layernorm_*).
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) rstd, y = xh gamma + beta
//   dx = rstd (t - mean(t) - xh mean(t xh)), t = dy gamma;   dgamma = sum_rows dy xh, dbeta = sum_rows dy
// All statistics and sums are f32; the variance is that of the centred values (no E[x^2] - mu^2 cancellation).
//
// About ten operations a value: bandwidth bounds both directions, so a row is read once and lives in registers (8 values x NV per lane) between the passes over it.  Rows up to 2048 wide
// belong to one wave (no barrier at all), rows up to 8192 to the four waves of a block; wider ones are read again for each pass and stay in the caches.
// Backward: one kernel reads x and dy once, writes dx and keeps this wave's part of dgamma and dbeta in registers over all its rows; the blocks' partial rows are then added in a
// fixed order.
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
constexpr int LN_PART = 512;          // blocks of the backward pass = partial rows of the parameter gradients

// sum over the W waves that share a row; `red` (W > 1) is reusable behind the next barrier
template <int W> __device__ __forceinline__ float ln_row_sum(float v, float* red) {
    v = wave_sum(v);
    if constexpr (W == 4) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (red[0] + red[1]) + (red[2] + red[3]);
    }
    return v;
}
}   // namespace

// W waves per row (1: four rows a block; 4: one), NV runs of 8 values per lane: D <= 512 W NV
template <typename T, int W, int NV>
__global__ __launch_bounds__(LN_THREADS) void ln_fwd_row_kernel(const T* __restrict__ x, long long ldx, long long M, int D, float eps, const float* __restrict__ gamma,
                                                                const float* __restrict__ beta, T* __restrict__ y, long long ldy, float* __restrict__ mean,
                                                                float* __restrict__ rstd) {
    __shared__ float red[2][4];
    const int lane = W == 1 ? (threadIdx.x & 63) : (int)threadIdx.x;
    const long long r = W == 1 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long long)blockIdx.x;
    if (r >= M) return;                                      // (W = 4: block-uniform)
    float f[NV][8];
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * W * 64 + lane) * 8;
        tok_ldn<T>(x + r * ldx + c, f[v], D - c);            // (0 past the row's end)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += f[v][i];
    }
    const float mu = ln_row_sum<W>(s, red[0]) / D;
    s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f[v][i] = (v * W * 64 + lane) * 8 + i < D ? f[v][i] - mu : 0.f;
            s += f[v][i] * f[v][i];
        }
    const float rs = 1.f / sqrtf(ln_row_sum<W>(s, red[1]) / D + eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * W * 64 + lane) * 8;
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

template <typename T, int W, int NV>
__global__ __launch_bounds__(LN_THREADS) void ln_bwd_row_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x, long long ldx, long long M, int D,
                                                                const float* __restrict__ gamma, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                T* __restrict__ dx, long long lddx, float* __restrict__ pg, float* __restrict__ pb) {
    __shared__ float red[2][2][4];
    __shared__ float acc[W == 1 ? 4 : 1][W == 1 ? 512 : 1];
    const int lane = W == 1 ? (threadIdx.x & 63) : (int)threadIdx.x, wave = threadIdx.x >> 6;
    const long long per = W == 1 ? 4 : 1;
    float g[NV][8], sg[NV][8], sb[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * W * 64 + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[v][i] = 1.f, sg[v][i] = sb[v][i] = 0.f;
        if (gamma != nullptr && c < D) tok_ldn<float>(gamma + c, g[v], D - c);
    }
    int flip = 0;
    for (long long r0 = blockIdx.x * per; r0 < M; r0 += gridDim.x * per) {
        const long long r = r0 + (W == 1 ? wave : 0);
        if (W == 1 && r >= M) break;                         // (this wave's last round; W = 4: block-uniform by the loop)
        const float mu = mean[r], rs = rstd[r];
        float f[NV][8], d[NV][8];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * W * 64 + lane) * 8;
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
            const float m1 = ln_row_sum<W>(s1, red[flip][0]) / D, m2 = ln_row_sum<W>(s2, red[flip][1]) / D;
            flip ^= 1;                                       // (the next round's sums go elsewhere: two barriers lie between two uses)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * W * 64 + lane) * 8;
                if (c < D) {
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = rs * (d[v][i] - m1 - f[v][i] * m2);
                    tok_stn<T>(dx + r * lddx + c, o, D - c);
                }
            }
        }
    }
    // this block's partial rows; the four waves of W = 1 are added in their order
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* const out = which == 0 ? pg : pb;
        if (out == nullptr) continue;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * W * 64 + lane) * 8;
            if constexpr (W == 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[wave][i * 64 + lane] = which == 0 ? sg[v][i] : sb[v][i];
                __syncthreads();
                for (int q = threadIdx.x; q < 512; q += LN_THREADS) {
                    const int i = q >> 6, l = q & 63, col = (v * 64 + l) * 8 + i;
                    if (col < D) out[(long long)blockIdx.x * D + col] = (acc[0][q] + acc[1][q]) + (acc[2][q] + acc[3][q]);
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
inline long long ln_rows(long long M) {
    long long r = 64;
    while ((M + r - 1) / r > 512) r *= 2;
    return r;
}
// waves per row and runs per lane that a width takes; 0: the kernels for any width
inline int ln_waves(int D) { return D <= 2048 ? 1 : (D <= 8192 ? 4 : 0); }
inline int ln_runs(int D) { return (D + 512 * ln_waves(D) - 1) / (512 * ln_waves(D)); }
inline long long ln_parts(long long M, int D) {
    const int w = ln_waves(D);
    if (w == 0) return (M + ln_rows(M) - 1) / ln_rows(M);
    const long long blocks = w == 1 ? (M + 3) / 4 : M;
    return blocks < LN_PART ? blocks : LN_PART;
}
template <typename T, typename F> int ln_by_width(int D, F&& f) {
    const int w = ln_waves(D), n = ln_runs(D);
    if (w == 1) {
        if (n == 1) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
        if (n == 2) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
        if (n == 3) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 3>{});
        return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
    }
    if (n == 2) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});          // (4 waves, 1 run: up to 2048, which one wave takes)
    if (n == 3) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 3>{});
    return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
}
template <typename T>
int ln_fwd(const void* x, long long ldx, long long M, int D, float eps, const float* gamma, const float* beta, void* y, long long ldy, float* mean, float* rstd, hipStream_t stream) {
    if (ln_waves(D) == 0) {
        hipLaunchKernelGGL((ln_fwd_kernel<T>), dim3((unsigned)M), dim3(LN_THREADS), 0, stream, (const T*)x, ldx, D, eps, gamma, beta, (T*)y, ldy, mean, rstd);
        return MIS_OK;
    }
    return ln_by_width<T>(D, [&](auto w, auto n) {
        constexpr int W = decltype(w)::value, NV = decltype(n)::value;
        hipLaunchKernelGGL((ln_fwd_row_kernel<T, W, NV>), dim3((unsigned)(W == 1 ? (M + 3) / 4 : M)), dim3(LN_THREADS), 0, stream, (const T*)x, ldx, M, D, eps, gamma, beta, (T*)y, ldy,
                           mean, rstd);
        return MIS_OK;
    });
}
template <typename T>
int ln_bwd(const void* dy, long long lddy, const void* x, long long ldx, long long M, int D, const float* gamma, const float* mean, const float* rstd, void* dx, long long lddx, float* pg,
           float* pb, hipStream_t stream) {
    const long long parts = ln_parts(M, D);
    if (ln_waves(D) == 0) {
        if (dx != nullptr)
            hipLaunchKernelGGL((ln_bwd_dx_kernel<T>), dim3((unsigned)M), dim3(LN_THREADS), 0, stream, (const T*)dy, lddy, (const T*)x, ldx, D, gamma, mean, rstd, (T*)dx, lddx);
        if (pg != nullptr || pb != nullptr)
            hipLaunchKernelGGL((ln_bwd_param_kernel<T>), dim3((unsigned)(parts * ((D + 63) / 64))), dim3(LN_THREADS), 0, stream, (const T*)dy, lddy, (const T*)x, ldx, M, D, mean, rstd, pg, pb,
                               ln_rows(M), (int)parts);
        return MIS_OK;
    }
    return ln_by_width<T>(D, [&](auto w, auto n) {
        constexpr int W = decltype(w)::value, NV = decltype(n)::value;
        hipLaunchKernelGGL((ln_bwd_row_kernel<T, W, NV>), dim3((unsigned)parts), dim3(LN_THREADS), 0, stream, (const T*)dy, lddy, (const T*)x, ldx, M, D, gamma, mean, rstd, (T*)dx, lddx, pg, pb);
        return MIS_OK;
    });
}
int ln_check(const char* who, int dtype, long long M, int D) {
    MIS_REQUIRE(dtype == MIS_F32 || dtype == MIS_BF16, MIS_EINVAL, "%s: dtype must be MIS_F32 or MIS_BF16", who);
    MIS_REQUIRE(M >= 0 && D >= 1, MIS_EINVAL, "%s: needs rows >= 0 and a width >= 1 (got %lld, %d)", who, M, D);
    MIS_REQUIRE(M < (1ll << 31), MIS_EUNSUPPORTED, "%s: %lld rows are more than a grid holds", who, M);
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
    if (dtype == MIS_BF16) ln_fwd<__bf16>(x, ldx, M, D, eps, gamma, beta, y, ldy, mean, rstd, s);
    else ln_fwd<float>(x, ldx, M, D, eps, gamma, beta, y, ldy, mean, rstd, s);
    MIS_LAUNCH_CHECK("mis_layernorm_fwd");
    return MIS_OK;
}

extern "C" size_t mis_layernorm_bwd_workspace_bytes(int dtype, long long M, int D) {
    if (ln_check("mis_layernorm_bwd", dtype, M, D) != MIS_OK || M == 0) return 0;
    return 2 * tok_align((size_t)ln_parts(M, D) * D * 4);
}

extern "C" int mis_layernorm_bwd(int dtype, const void* dy, long long lddy, const void* x, long long ldx, long long M, int D, const float* gamma, const float* mean,
                                 const float* rstd, void* dx, long long lddx, float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes, void* stream_) {
    const hipStream_t stream = (hipStream_t)stream_;
    if (const int rc = ln_check("mis_layernorm_bwd", dtype, M, D)) return rc;
    MIS_REQUIRE(M == 0 || (dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr), MIS_EINVAL, "mis_layernorm_bwd: null pointer");
    MIS_REQUIRE(lddy >= D && ldx >= D && (dx == nullptr || lddx >= D), MIS_EINVAL, "mis_layernorm_bwd: a row stride is below the width");
    const long long parts = M > 0 ? ln_parts(M, D) : 0;
    const bool params = dgamma != nullptr || dbeta != nullptr;
    const size_t half = tok_align((size_t)parts * D * 4);
    MIS_REQUIRE(!params || M == 0 || (workspace != nullptr && workspace_bytes >= 2 * half), MIS_EINVAL, "mis_layernorm_bwd: the workspace has %zu bytes, %zu are needed",
                workspace_bytes, 2 * half);
    float* const pg = dgamma != nullptr ? (float*)workspace : nullptr;
    float* const pb = dbeta != nullptr ? (float*)((char*)workspace + half) : nullptr;
    if (M > 0 && (params || dx != nullptr)) {
        if (dtype == MIS_BF16) ln_bwd<__bf16>(dy, lddy, x, ldx, M, D, gamma, mean, rstd, dx, lddx, pg, pb, stream);
        else ln_bwd<float>(dy, lddy, x, ldx, M, D, gamma, mean, rstd, dx, lddx, pg, pb, stream);
        MIS_LAUNCH_CHECK("mis_layernorm_bwd");
    }
    // (no rows: the sums are over nothing and the gradients zero)
    if (params) return tok_column_sums(pg, pb, parts, D, dgamma, dbeta, stream);
    return MIS_OK;
}
