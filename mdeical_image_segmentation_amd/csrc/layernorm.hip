// Layer norm over the channels of a token, forward and backward (include/misamd.h: mis_layernorm_*).
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) rstd, y = xh gamma + beta
//   dx = rstd (t - mean(t) - xh mean(t xh)), t = dy gamma;   dgamma = sum_rows dy xh, dbeta = sum_rows dy
// All statistics and sums are f32; the variance is that of the centred values (no E[x^2] - mu^2 cancellation).
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

__global__ __launch_bounds__(256) void ln_param_sum_kernel(const float* __restrict__ pg, const float* __restrict__ pb, long long nrow, int D, float* __restrict__ dgamma,
                                                           float* __restrict__ dbeta) {
    __shared__ float red[4][64];
    const float* const part = blockIdx.y == 0 ? pg : pb;
    float* const out = blockIdx.y == 0 ? dgamma : dbeta;
    if (out == nullptr) return;                              // (block-uniform)
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6;
    const long long n = (long long)blockIdx.x * 64 + c;
    float s = 0.f;
    if (n < D)
        for (long long r = g; r < nrow; r += 4) s += part[r * D + n];
    red[g][c] = s;
    __syncthreads();
    if (g == 0 && n < D) out[n] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
}

namespace {
inline long long ln_rows(long long M) {
    long long r = 64;
    while ((M + r - 1) / r > 512) r *= 2;
    return r;
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
    if (dtype == MIS_BF16)
        hipLaunchKernelGGL((ln_fwd_kernel<__bf16>), dim3((unsigned)M), dim3(LN_THREADS), 0, (hipStream_t)stream, (const __bf16*)x, ldx, D, eps, gamma, beta, (__bf16*)y, ldy, mean, rstd);
    else
        hipLaunchKernelGGL((ln_fwd_kernel<float>), dim3((unsigned)M), dim3(LN_THREADS), 0, (hipStream_t)stream, (const float*)x, ldx, D, eps, gamma, beta, (float*)y, ldy, mean, rstd);
    MIS_LAUNCH_CHECK("mis_layernorm_fwd");
    return MIS_OK;
}

extern "C" size_t mis_layernorm_bwd_workspace_bytes(int dtype, long long M, int D) {
    if (ln_check("mis_layernorm_bwd", dtype, M, D) != MIS_OK || M == 0) return 0;
    return 2 * tok_align((size_t)((M + ln_rows(M) - 1) / ln_rows(M)) * D * 4);
}

extern "C" int mis_layernorm_bwd(int dtype, const void* dy, long long lddy, const void* x, long long ldx, long long M, int D, const float* gamma, const float* mean,
                                 const float* rstd, void* dx, long long lddx, float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes, void* stream_) {
    const hipStream_t stream = (hipStream_t)stream_;
    if (const int rc = ln_check("mis_layernorm_bwd", dtype, M, D)) return rc;
    MIS_REQUIRE(M == 0 || (dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr), MIS_EINVAL, "mis_layernorm_bwd: null pointer");
    MIS_REQUIRE(lddy >= D && ldx >= D && (dx == nullptr || lddx >= D), MIS_EINVAL, "mis_layernorm_bwd: a row stride is below the width");
    const long long rows = ln_rows(M), nrb = (M + rows - 1) / rows;
    const bool params = dgamma != nullptr || dbeta != nullptr;
    const size_t half = tok_align((size_t)nrb * D * 4);
    MIS_REQUIRE(!params || M == 0 || (workspace != nullptr && workspace_bytes >= 2 * half), MIS_EINVAL, "mis_layernorm_bwd: the workspace has %zu bytes, %zu are needed",
                workspace_bytes, 2 * half);
    float* const pg = (float*)workspace;
    float* const pb = (float*)((char*)workspace + half);
    if (dx != nullptr && M > 0) {
        if (dtype == MIS_BF16)
            hipLaunchKernelGGL((ln_bwd_dx_kernel<__bf16>), dim3((unsigned)M), dim3(LN_THREADS), 0, stream, (const __bf16*)dy, lddy, (const __bf16*)x, ldx, D, gamma, mean, rstd, (__bf16*)dx, lddx);
        else
            hipLaunchKernelGGL((ln_bwd_dx_kernel<float>), dim3((unsigned)M), dim3(LN_THREADS), 0, stream, (const float*)dy, lddy, (const float*)x, ldx, D, gamma, mean, rstd, (float*)dx, lddx);
        MIS_LAUNCH_CHECK("mis_layernorm_bwd (dx)");
    }
    if (params) {
        if (M > 0) {
            const dim3 grid((unsigned)(nrb * ((D + 63) / 64)));
            if (dtype == MIS_BF16)
                hipLaunchKernelGGL((ln_bwd_param_kernel<__bf16>), grid, dim3(LN_THREADS), 0, stream, (const __bf16*)dy, lddy, (const __bf16*)x, ldx, M, D, mean, rstd, pg, pb, rows, (int)nrb);
            else
                hipLaunchKernelGGL((ln_bwd_param_kernel<float>), grid, dim3(LN_THREADS), 0, stream, (const float*)dy, lddy, (const float*)x, ldx, M, D, mean, rstd, pg, pb, rows, (int)nrb);
            MIS_LAUNCH_CHECK("mis_layernorm_bwd (partial sums)");
        }
        // (no rows: the sums are over nothing and the gradients zero)
        hipLaunchKernelGGL(ln_param_sum_kernel, dim3((unsigned)((D + 63) / 64), 2), dim3(256), 0, stream, pg, pb, nrb, D, dgamma, dbeta);
        MIS_LAUNCH_CHECK("mis_layernorm_bwd (sums)");
    }
    return MIS_OK;
}
