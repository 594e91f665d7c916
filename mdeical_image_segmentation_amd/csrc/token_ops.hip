// C entries of the token operators' matrix products (include/misamd.h: mis_linear_*, mis_gated_ffn_*) and the element-wise part of their backward passes.
//
//   linear:  z = x W^T + b, y = act(z) + res          dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum_rows dz
//   gated:   g = x Wg^T + bg, u = x Wu^T + bu,        dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, biases: row sums of dg, du
//            h = act(g) u
// What a forward pass keeps: the pre-activations in f32, whatever the type.  The bias gradients are f32 sums of dz, and 2^-9 in every term would show in them; and a form of fewer bits that
// neighbouring columns share an exponent in (8 values in 16 bytes: 32768 x 1024 x 2 x 4096 training 1724 us instead of 1858) costs a column that is small beside its neighbours its
// gradient.  dz (dg | du) is rounded to the operand type once, for the matrix instructions; the bias sums are taken before that rounding, per block of rows, and the blocks' partial rows are
// added in a fixed order.
#include "tok_gemm.hpp"

namespace {
constexpr int TO_COLS = 128;          // columns of a block (16 threads x 8)
// rows of a block: 64, more when that would leave over 512 partial rows for the second pass (32768 x 4096 bf16 with a bias: 512 partial rows 152 us, 128 of them 139; 16384 x 1024 20 / 19;
// with 128 a narrow gradient of many rows is too few blocks)
inline long long to_rows(long long M) {
    long long r = 64;
    while ((M + r - 1) / r > 512) r *= 2;
    return r;
}
inline long long to_nblk(long long M) { return (M + to_rows(M) - 1) / to_rows(M); }
}   // namespace

// Bandwidth: per value 2 bytes of dy, 4 of z, 2 of dz; gated twice the last two.  32768 x 4096 gated bf16: 1.9 GB in 414 us, 4.5 TB/s.
// dz = dy act'(z) (MODE 0: linear), (dg | du) (MODE 1: gated), nothing but the column sums of dy (MODE 2).  A thread: 8 columns, every 16th row of its block.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void tok_dz_kernel(const T* __restrict__ dy, long long lddy, const float* __restrict__ kept, const float* __restrict__ kept2, int act, long long M, long long N, T* __restrict__ dz, long long lddz, float* __restrict__ part, float* __restrict__ part2,
                                                     long long rows, int nrb) {
    constexpr bool PRECISE = sizeof(T) == 4;
    __shared__ float red[2][16][TO_COLS];
    const int cg = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const long long rb = blockIdx.x % nrb, n = (long long)(blockIdx.x / nrb) * TO_COLS + cg * 8;
    const int nv = N - n >= 8 ? 8 : (N > n ? (int)(N - n) : 0);
    float s[8], s2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = s2[i] = 0.f;
    const long long m1 = (rb + 1) * rows < M ? (rb + 1) * rows : M;
    if (nv > 0)
        for (long long m = rb * rows + rl; m < m1; m += 16) {
            float d[8];
            tok_ldn<T>(dy + m * lddy + n, d, nv);
            if constexpr (MODE == 0) {
                float v[8], e[8];
                tok_ldn<float>(kept + m * N + n, v, nv);
                tok_act8<PRECISE, true>(act, v, e);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= e[i];
                if (dz != nullptr) tok_st8<T>(dz + m * lddz + n, d);          // (a row's pitch is whole runs of 8; behind column N: zeros)
            } else if constexpr (MODE == 1) {
                float g[8], e[8], u[8], du[8];
                tok_ldn<float>(kept + m * N + n, g, nv);
                tok_ldn<float>(kept2 + m * N + n, u, nv);
                tok_act8<PRECISE, true>(act, g, e);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    du[i] = d[i] * g[i];
                    d[i] = d[i] * (e[i] * u[i]);
                    s2[i] += du[i];
                }
                tok_st8<T>(dz + m * lddz + n, d);
                tok_st8<T>(dz + m * lddz + (lddz >> 1) + n, du);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += d[i];
        }
    if (part == nullptr && part2 == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        red[0][rl][cg * 8 + i] = s[i];
        if constexpr (MODE == 1) red[1][rl][cg * 8 + i] = s2[i];
    }
    __syncthreads();
    const int w = threadIdx.x >> 7, c = threadIdx.x & 127;          // first 128 threads: s, the others: s2
    const long long col = (long long)(blockIdx.x / nrb) * TO_COLS + c;
    float* const out = w == 0 ? part : part2;
    if ((w == 0 || MODE == 1) && out != nullptr && col < N) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) t += red[w][r][c];
        out[rb * N + col] = t;
    }
}

// Up to three matrices, `cols` values a row, rows ld apart -> the same rows at a pitch of whole runs of 8, zeros behind them
struct ToPack {
    struct { const void* src; long long ld, rows, cols; void* dst; } m[3];
};
template <typename T> __global__ __launch_bounds__(256) void tok_pack_kernel(const ToPack p) {
    const T* const src = reinterpret_cast<const T*>(blockIdx.y == 0 ? p.m[0].src : blockIdx.y == 1 ? p.m[1].src : p.m[2].src);
    T* const dst = reinterpret_cast<T*>(blockIdx.y == 0 ? p.m[0].dst : blockIdx.y == 1 ? p.m[1].dst : p.m[2].dst);
    const long long ld = blockIdx.y == 0 ? p.m[0].ld : blockIdx.y == 1 ? p.m[1].ld : p.m[2].ld, rows = blockIdx.y == 0 ? p.m[0].rows : blockIdx.y == 1 ? p.m[1].rows : p.m[2].rows,
                    cols = blockIdx.y == 0 ? p.m[0].cols : blockIdx.y == 1 ? p.m[1].cols : p.m[2].cols;
    const long long per = (cols + 7) >> 3, pitch = per * 8;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (long long)gridDim.x * 256) {
        const long long r = i / per, c = (i - r * per) * 8;
        float v[8];
        tok_ldn<T>(src + r * ld + c, v, cols - c >= 8 ? 8 : (int)(cols - c));
        tok_st8<T>(dst + r * pitch + c, v);
    }
}

// Column sums of up to a few hundred partial rows: 16 row groups a block, so that a thread adds some 32 values with 8 loads in flight (four groups of 256 threads took 39 us for
// 512 x 1024 partial rows, this one 5)
__global__ __launch_bounds__(1024) void tok_colsum_kernel(const float* __restrict__ p0, const float* __restrict__ p1, long long nrow, long long N, long long col0,
                                                          float* __restrict__ out0, float* __restrict__ out1) {
    __shared__ float red[16][64];
    const float* const part = blockIdx.y == 0 ? p0 : p1;
    float* const out = blockIdx.y == 0 ? out0 : out1;
    if (out == nullptr) return;                              // (block-uniform)
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6;
    const long long n = (col0 + blockIdx.x) * 64 + c;
    float s = 0.f;
    if (n < N) {
        long long r = g;
        for (; r + 7 * 16 < nrow; r += 8 * 16) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = part[(r + i * 16) * N + n];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; r < nrow; r += 16) s += part[r * N + n];
    }
    red[g][c] = s;
    __syncthreads();
    if (g == 0 && n < N) {
#pragma unroll
        for (int q = 1; q < 16; ++q) s += red[q][c];
        out[n] = s;
    }
}

int tok_column_sums(const float* p0, const float* p1, long long nrow, long long N, float* out0, float* out1, hipStream_t stream) {
    constexpr long long most = TOK_BLOCKS / 8;          // (2 x 1024 threads for 64 columns: 2^27 columns at a time)
    for (long long col0 = 0, all = (N + 63) / 64; col0 < all; col0 += most) {
        hipLaunchKernelGGL(tok_colsum_kernel, dim3((unsigned)(all - col0 < most ? all - col0 : most), out1 != nullptr ? 2 : 1), dim3(1024), 0, stream, p0, p1, nrow, N, col0, out0, out1);
        MIS_LAUNCH_CHECK("token column sums");
    }
    return MIS_OK;
}

namespace {
// bytes of one [M][N] tensor that a forward pass keeps
size_t kept_of(long long M, long long N) { return tok_align((size_t)M * N * 4); }
template <int MODE>
int to_dz(int dtype, const void* dy, long long lddy, const void* kept, int act, long long M, long long N, void* dz, long long lddz, float* part, float* part2,
          hipStream_t stream) {
    const long long rows = to_rows(M), nrb = to_nblk(M), ncb = (N + TO_COLS - 1) / TO_COLS;
    MIS_REQUIRE(nrb * ncb < TOK_BLOCKS, MIS_EUNSUPPORTED, "token gradient: the grid is too large");
    const dim3 grid((unsigned)(nrb * ncb));
    const float *k0 = (const float*)kept, *k1 = MODE == 1 ? (const float*)((const char*)kept + kept_of(M, N)) : nullptr;
    if (dtype == MIS_BF16)
        hipLaunchKernelGGL((tok_dz_kernel<__bf16, MODE>), grid, dim3(256), 0, stream, (const __bf16*)dy, lddy, k0, k1, act, M, N, (__bf16*)dz, lddz, part, part2, rows, (int)nrb);
    else
        hipLaunchKernelGGL((tok_dz_kernel<float, MODE>), grid, dim3(256), 0, stream, (const float*)dy, lddy, k0, k1, act, M, N, (float*)dz, lddz, part, part2, rows, (int)nrb);
    MIS_LAUNCH_CHECK("token gradient");
    return MIS_OK;
}
// row pitch of copies and of dz: whole runs of 8, so that the products read 16-byte chunks whatever the width is
inline long long to_pitch(long long n) { return (n + 7) / 8 * 8; }
inline size_t es_of(int dtype) { return dtype == MIS_BF16 ? 2 : 4; }

constexpr long long TO_MAX = 1ll << 40;          // elements of one tensor: keeps every byte offset and workspace size far inside 64 bits

int check_dims(const char* who, int dtype, int act, long long M, int N, int K) {
    MIS_REQUIRE(dtype == MIS_F32 || dtype == MIS_BF16, MIS_EINVAL, "%s: dtype must be MIS_F32 or MIS_BF16", who);
    MIS_REQUIRE(tok_act_ok(act), MIS_EINVAL, "%s: unknown activation %d", who, act);
    MIS_REQUIRE(M >= 0 && N >= 1 && K >= 1, MIS_EINVAL, "%s: needs rows >= 0 and widths >= 1 (got %lld, %d, %d)", who, M, N, K);
    MIS_REQUIRE(M < (1ll << 31) && M < TO_MAX / N && M < TO_MAX / K, MIS_EUNSUPPORTED, "%s: %lld rows of %d / %d values are too many", who, M, N, K);
    return MIS_OK;
}
#define TO_LD(who, ld, n, what) MIS_REQUIRE((ld) >= (n) && (ld) < TO_MAX, MIS_EINVAL, "%s: the row stride of " what " (%lld) is below its width", who, (long long)(ld))
#define TO_PTR(who, p, what) MIS_REQUIRE((p) != nullptr, MIS_EINVAL, "%s: " what " is null", who)

// Products want operands whose rows start on 16 bytes and end on whole chunks.  In a backward pass whose products are large enough to pay for a copy the others are copied to such rows first.
// dx and dW of an odd-sized linear, M x K x N, us with copies / without (dz and (dg | du) lie so from the start):
//                                bf16              f32        (dx alone: bf16    f32)
//      251 x 257 x 255          18 / 18           21 / 24            14 / 10   14 / 11
//      411 x 405 x 403          19 / 28           31 / 36            14 / 12   17 / 18
//      640 x 637 x 651          21 / 37           35 / 35            14 / 17   21 / 20
//      1023 x 1021 x 1027       34 / 64           71 / 82            17 / 24   37 / 38
//      1531 x 717 x 1209        38 / 81           88 / 108           22 / 30   49 / 51
//      2047 x 2049 x 2051       95 / 181         404 / 443           50 / 81  209 / 223
//      4099 x 1027 x 4097      134 / 434         757 / 860           74 / 205 387 / 429
constexpr double TO_PACK = 1 << 26;          // multiply-adds of a product from which on a copy pays
bool whole(const void* p, long long ld, long long n, size_t es) { return ((uintptr_t)p | (size_t)(ld * (long long)es)) % 16 == 0 && n % (16 / (long long)es) == 0; }
struct LinWs {
    bool act, pack_dy, pack_w, pack_x;
    size_t dz, w, x, part, slab_x, slab_w, total;
};
LinWs lin_ws(const MisLinearDesc* d) {
    LinWs w{};
    size_t at = 0;
    const size_t es = es_of(d->dtype);
    const bool large = (double)d->M * d->N * d->K >= TO_PACK, prod = d->dx != nullptr || d->dw != nullptr;
    w.act = d->act != MIS_ACT_NONE;
    w.pack_dy = !w.act && prod && large && !whole(d->dy, d->lddy, d->N, es);
    w.pack_w = d->dx != nullptr && large && !whole(d->w, d->ldw, d->K, es);
    w.pack_x = d->dw != nullptr && large && !whole(d->x, d->ldx, d->K, es);
    w.dz = at;
    if ((w.act && prod) || w.pack_dy) at += tok_align((size_t)d->M * to_pitch(d->N) * es);
    w.w = at;
    if (w.pack_w) at += tok_align((size_t)d->N * to_pitch(d->K) * es);
    w.x = at;
    if (w.pack_x) at += tok_align((size_t)d->M * to_pitch(d->K) * es);
    w.part = at;
    if (d->dbias != nullptr) at += tok_align((size_t)to_nblk(d->M) * d->N * 4);
    w.slab_x = at;
    if (d->dx != nullptr) at += tg_slab_bytes(d->dtype, TG_STORE, d->M, d->K, d->N, 1, 1);
    w.slab_w = at;
    if (d->dw != nullptr) at += tg_slab_bytes(d->dtype, TG_STORE, d->N, d->K, d->M, 1, 1);
    w.total = at;
    return w;
}
struct GatWs {
    bool pack_w, pack_x;
    size_t dz, w, x, pg, pu, slab_x, slab_w, total;
};
GatWs gat_ws(const MisGatedDesc* d) {
    GatWs w{};
    size_t at = 0;
    const size_t es = es_of(d->dtype);
    const bool large = (double)d->M * d->F * d->K >= TO_PACK;
    w.pack_w = d->dx != nullptr && large && !(whole(d->wg, d->ldw, d->K, es) && whole(d->wu, d->ldw, d->K, es));
    w.pack_x = d->dwg != nullptr && large && !whole(d->x, d->ldx, d->K, es);
    w.dz = at;
    at += tok_align((size_t)d->M * 2 * to_pitch(d->F) * es);
    w.w = at;
    if (w.pack_w) at += 2 * tok_align((size_t)d->F * to_pitch(d->K) * es);
    w.x = at;
    if (w.pack_x) at += tok_align((size_t)d->M * to_pitch(d->K) * es);
    w.pg = at;
    if (d->dbg != nullptr) at += tok_align((size_t)to_nblk(d->M) * d->F * 4);
    w.pu = at;
    if (d->dbu != nullptr) at += tok_align((size_t)to_nblk(d->M) * d->F * 4);
    w.slab_x = at;
    if (d->dx != nullptr) at += tg_slab_bytes(d->dtype, TG_STORE, d->M, d->K, d->F, 2, 1);
    w.slab_w = at;
    if (d->dwg != nullptr) at += tg_slab_bytes(d->dtype, TG_STORE, d->F, d->K, d->M, 1, 2);
    w.total = at;
    return w;
}
// the copies of a call, enqueued together
struct ToCopies {
    ToPack p{};
    int n = 0;
    long long runs = 0;          // of the largest
    TgOperand add(const void* src, long long ld, long long rows, long long cols, void* dst) {
        p.m[n].src = src; p.m[n].ld = ld; p.m[n].rows = rows; p.m[n].cols = cols; p.m[n].dst = dst;
        ++n;
        const long long r = rows * (to_pitch(cols) / 8);
        runs = r > runs ? r : runs;
        return TgOperand{dst, dst, to_pitch(cols), true};
    }
    int go(int dtype, hipStream_t stream) const {
        if (n == 0) return MIS_OK;
        const long long b = (runs + 255) / 256;
        const dim3 grid((unsigned)(b < 8192 ? b : 8192), (unsigned)n);
        if (dtype == MIS_BF16) hipLaunchKernelGGL(tok_pack_kernel<__bf16>, grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL(tok_pack_kernel<float>, grid, dim3(256), 0, stream, p);
        MIS_LAUNCH_CHECK("token rows");
        return MIS_OK;
    }
};
// an empty batch has zero gradients
__global__ void tok_zero_kernel(char* p, long long pitch, long long rows, long long bytes) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < rows * bytes; i += (long long)gridDim.x * blockDim.x) p[(i / bytes) * pitch + i % bytes] = 0;
}
int to_zero(void* p, long long ld, long long rows, long long cols, size_t es, hipStream_t s) {
    const long long n = rows * cols * (long long)es;
    hipLaunchKernelGGL(tok_zero_kernel, dim3((unsigned)(n < (1 << 20) ? (n + 255) / 256 : 4096)), dim3(256), 0, s, (char*)p, ld * (long long)es, rows, cols * (long long)es);
    MIS_LAUNCH_CHECK("token zero");
    return MIS_OK;
}
#define TO_TRY(call)                       \
    do {                                   \
        if (const int rc__ = (call)) return rc__; \
    } while (0)
}   // namespace

extern "C" size_t mis_linear_kept_bytes(const MisLinearDesc* d) {
    if (d == nullptr || check_dims("mis_linear", d->dtype, d->act, d->M, d->N, d->K) != MIS_OK || d->act == MIS_ACT_NONE) return 0;
    return kept_of(d->M, d->N);
}

extern "C" size_t mis_linear_fwd_workspace_bytes(const MisLinearDesc* d) {
    if (d == nullptr || check_dims("mis_linear_fwd", d->dtype, d->act, d->M, d->N, d->K) != MIS_OK) return 0;
    return tg_slab_bytes(d->dtype, TG_LINEAR, d->M, d->N, d->K, 1, 1);
}

extern "C" int mis_linear_fwd(const MisLinearDesc* d, void* stream_) {
    const hipStream_t stream = (hipStream_t)stream_;
    const char* who = "mis_linear_fwd";
    TO_PTR(who, d, "the descriptor");
    TO_TRY(check_dims(who, d->dtype, d->act, d->M, d->N, d->K));
    if (d->M == 0) return MIS_OK;
    TO_PTR(who, d->x, "x"); TO_PTR(who, d->w, "w"); TO_PTR(who, d->y, "y");
    TO_LD(who, d->ldx, d->K, "x"); TO_LD(who, d->ldw, d->K, "w"); TO_LD(who, d->ldy, d->N, "y");
    if (d->res != nullptr) TO_LD(who, d->ldres, d->N, "res");
    MIS_REQUIRE((uintptr_t)d->kept % 16 == 0, MIS_EINVAL, "%s: kept must be 16-byte aligned", who);
    TgArgs a{};
    a.ranges = a.batches = 1;
    a.a = TgOperand{d->x, d->x, d->ldx, false};
    a.b = TgOperand{d->w, d->w, d->ldw, false};
    a.M = d->M; a.N = d->N; a.K = d->K;
    a.act = d->act; a.bias = d->bias; a.res = d->res; a.ldres = d->ldres;
    a.y = a.y2 = d->y; a.ldy = d->ldy;
    if (d->act != MIS_ACT_NONE) a.kept = (float*)d->kept;
    const size_t need = mis_linear_fwd_workspace_bytes(d);
    return tg_launch(d->dtype, 0, 0, TG_LINEAR, a, need > 0 && d->workspace != nullptr && d->workspace_bytes >= need ? (float*)d->workspace : nullptr, stream);
}

extern "C" size_t mis_linear_bwd_workspace_bytes(const MisLinearDesc* d) {
    if (d == nullptr || check_dims("mis_linear_bwd", d->dtype, d->act, d->M, d->N, d->K) != MIS_OK) return 0;
    return lin_ws(d).total;
}

extern "C" int mis_linear_bwd(const MisLinearDesc* d, void* stream_) {
    const hipStream_t stream = (hipStream_t)stream_;
    const char* who = "mis_linear_bwd";
    TO_PTR(who, d, "the descriptor");
    TO_TRY(check_dims(who, d->dtype, d->act, d->M, d->N, d->K));
    const size_t es = es_of(d->dtype);
    if (d->dw != nullptr) TO_LD(who, d->lddw, d->K, "dw");
    if (d->M == 0) {
        if (d->dw != nullptr) TO_TRY(to_zero(d->dw, d->lddw, d->N, d->K, es, stream));
        if (d->dbias != nullptr) TO_TRY(to_zero(d->dbias, d->N, 1, d->N, 4, stream));
        return MIS_OK;
    }
    const bool act = d->act != MIS_ACT_NONE, prod = d->dx != nullptr || d->dw != nullptr;
    TO_PTR(who, d->dy, "dy");
    TO_LD(who, d->lddy, d->N, "dy");
    if (act) {
        TO_PTR(who, d->kept, "what the forward pass keeps");
        MIS_REQUIRE((uintptr_t)d->kept % 16 == 0, MIS_EINVAL, "%s: kept must be 16-byte aligned", who);
        MIS_REQUIRE(d->dbias == nullptr || d->bias != nullptr || d->dtype == MIS_F32, MIS_EINVAL, "%s: dbias without bias", who);          // (f32 calls may have it alone)
    }
    if (d->dx != nullptr) { TO_PTR(who, d->w, "w"); TO_LD(who, d->ldw, d->K, "w"); TO_LD(who, d->lddx, d->K, "dx"); }
    if (d->dw != nullptr) { TO_PTR(who, d->x, "x"); TO_LD(who, d->ldx, d->K, "x"); }
    const LinWs w = lin_ws(d);
    MIS_REQUIRE(w.total == 0 || (d->workspace != nullptr && d->workspace_bytes >= w.total), MIS_EINVAL, "%s: the workspace has %zu bytes, %zu are needed", who, d->workspace_bytes, w.total);
    char* const ws = (char*)d->workspace;
    TgOperand dz{d->dy, d->dy, d->lddy, false};
    float* const part = d->dbias != nullptr ? (float*)(ws + w.part) : nullptr;
    ToCopies copies;
    if (w.act) {
        dz = TgOperand{ws + w.dz, ws + w.dz, to_pitch(d->N), true};
        if (prod || part != nullptr)
            TO_TRY(to_dz<0>(d->dtype, d->dy, d->lddy, d->kept, d->act, d->M, d->N, prod ? ws + w.dz : nullptr, dz.ld, part, nullptr, stream));
    } else {
        if (part != nullptr) TO_TRY(to_dz<2>(d->dtype, d->dy, d->lddy, nullptr, 0, d->M, d->N, nullptr, 0, part, nullptr, stream));
        if (w.pack_dy) dz = copies.add(d->dy, d->lddy, d->M, d->N, ws + w.dz);
    }
    if (part != nullptr) TO_TRY(tok_column_sums(part, nullptr, to_nblk(d->M), d->N, d->dbias, nullptr, stream));
    TgOperand W{d->w, d->w, d->ldw, false}, X{d->x, d->x, d->ldx, false};
    if (w.pack_w) W = copies.add(d->w, d->ldw, d->N, d->K, ws + w.w);
    if (w.pack_x) X = copies.add(d->x, d->ldx, d->M, d->K, ws + w.x);
    TO_TRY(copies.go(d->dtype, stream));
    TgSum sx{}, sw{};
    if (d->dx != nullptr) {
        TgArgs a{};
        a.ranges = a.batches = 1;
        a.a = dz;
        a.b = W;
        a.M = d->M; a.N = d->K; a.K = d->N;
        a.y = a.y2 = d->dx; a.ldy = d->lddx;
        TO_TRY(tg_launch(d->dtype, 0, 1, TG_STORE, a, (float*)(ws + w.slab_x), stream, &sx));
    }
    if (d->dw != nullptr) {
        TgArgs a{};
        a.ranges = a.batches = 1;
        a.a = dz;
        a.b = X;
        a.M = d->N; a.N = d->K; a.K = d->M;
        a.y = a.y2 = d->dw; a.ldy = d->lddw;
        TO_TRY(tg_launch(d->dtype, 1, 1, TG_STORE, a, (float*)(ws + w.slab_w), stream, &sw));
    }
    return tg_sums(d->dtype, sx, sw, stream);
}

extern "C" size_t mis_gated_ffn_kept_bytes(const MisGatedDesc* d) {
    if (d == nullptr || check_dims("mis_gated_ffn", d->dtype, d->act, d->M, d->F, d->K) != MIS_OK) return 0;
    return 2 * kept_of(d->M, d->F);
}

extern "C" size_t mis_gated_ffn_fwd_workspace_bytes(const MisGatedDesc* d) {
    if (d == nullptr || check_dims("mis_gated_ffn_fwd", d->dtype, d->act, d->M, d->F, d->K) != MIS_OK) return 0;
    return tg_slab_bytes(d->dtype, TG_GATED, d->M, d->F, d->K, 1, 1);
}

extern "C" int mis_gated_ffn_fwd(const MisGatedDesc* d, void* stream_) {
    const hipStream_t stream = (hipStream_t)stream_;
    const char* who = "mis_gated_ffn_fwd";
    TO_PTR(who, d, "the descriptor");
    TO_TRY(check_dims(who, d->dtype, d->act, d->M, d->F, d->K));
    if (d->M == 0) return MIS_OK;
    TO_PTR(who, d->x, "x"); TO_PTR(who, d->wg, "wg"); TO_PTR(who, d->wu, "wu"); TO_PTR(who, d->h, "h");
    TO_LD(who, d->ldx, d->K, "x"); TO_LD(who, d->ldw, d->K, "wg / wu"); TO_LD(who, d->ldh, d->F, "h");
    MIS_REQUIRE((uintptr_t)d->kept % 16 == 0, MIS_EINVAL, "%s: kept must be 16-byte aligned", who);
    TgArgs a{};
    a.ranges = a.batches = 1;
    a.a = TgOperand{d->x, d->x, d->ldx, false};
    a.b = TgOperand{d->wg, d->wu, d->ldw, false};
    a.M = d->M; a.N = d->F; a.K = d->K;
    a.act = d->act; a.bias = d->bg; a.bias2 = d->bu;
    a.y = a.y2 = d->h; a.ldy = d->ldh;
    if (d->kept != nullptr) {
        a.kept = (float*)d->kept;
        a.kept2 = (float*)((char*)d->kept + kept_of(d->M, d->F));
    }
    const size_t need = mis_gated_ffn_fwd_workspace_bytes(d);
    return tg_launch(d->dtype, 0, 0, TG_GATED, a, need > 0 && d->workspace != nullptr && d->workspace_bytes >= need ? (float*)d->workspace : nullptr, stream);
}

extern "C" size_t mis_gated_ffn_bwd_workspace_bytes(const MisGatedDesc* d) {
    if (d == nullptr || check_dims("mis_gated_ffn_bwd", d->dtype, d->act, d->M, d->F, d->K) != MIS_OK) return 0;
    return gat_ws(d).total;
}

extern "C" int mis_gated_ffn_bwd(const MisGatedDesc* d, void* stream_) {
    const hipStream_t stream = (hipStream_t)stream_;
    const char* who = "mis_gated_ffn_bwd";
    TO_PTR(who, d, "the descriptor");
    TO_TRY(check_dims(who, d->dtype, d->act, d->M, d->F, d->K));
    const size_t es = es_of(d->dtype);
    MIS_REQUIRE((d->dwg == nullptr) == (d->dwu == nullptr), MIS_EINVAL, "%s: dwg and dwu come together", who);
    if (d->dwg != nullptr) TO_LD(who, d->lddw, d->K, "dwg / dwu");
    if (d->M == 0) {
        if (d->dwg != nullptr) {
            TO_TRY(to_zero(d->dwg, d->lddw, d->F, d->K, es, stream));
            TO_TRY(to_zero(d->dwu, d->lddw, d->F, d->K, es, stream));
        }
        if (d->dbg != nullptr) TO_TRY(to_zero(d->dbg, d->F, 1, d->F, 4, stream));
        if (d->dbu != nullptr) TO_TRY(to_zero(d->dbu, d->F, 1, d->F, 4, stream));
        return MIS_OK;
    }
    TO_PTR(who, d->dh, "dh"); TO_PTR(who, d->kept, "what the forward pass keeps");
    TO_LD(who, d->lddh, d->F, "dh");
    MIS_REQUIRE((uintptr_t)d->kept % 16 == 0, MIS_EINVAL, "%s: kept must be 16-byte aligned", who);
    MIS_REQUIRE((d->dbg == nullptr && d->dbu == nullptr) || d->bg != nullptr || d->bu != nullptr || d->dtype == MIS_F32, MIS_EINVAL, "%s: dbg / dbu without bg / bu", who);
    if (d->dx != nullptr) {
        TO_PTR(who, d->wg, "wg"); TO_PTR(who, d->wu, "wu");
        TO_LD(who, d->ldw, d->K, "wg / wu"); TO_LD(who, d->lddx, d->K, "dx");
    }
    if (d->dwg != nullptr) { TO_PTR(who, d->x, "x"); TO_LD(who, d->ldx, d->K, "x"); }
    const GatWs w = gat_ws(d);
    MIS_REQUIRE(d->workspace != nullptr && d->workspace_bytes >= w.total, MIS_EINVAL, "%s: the workspace has %zu bytes, %zu are needed", who, d->workspace_bytes, w.total);
    char* const ws = (char*)d->workspace;
    const long long F = d->F, pitch = to_pitch(F), lddz = 2 * pitch;
    float* const pg = d->dbg != nullptr ? (float*)(ws + w.pg) : nullptr;
    float* const pu = d->dbu != nullptr ? (float*)(ws + w.pu) : nullptr;
    void* const dz = ws + w.dz;          // [M][dg (F, padded to pitch) | du]
    void* const du = ws + w.dz + pitch * es;
    TO_TRY(to_dz<1>(d->dtype, d->dh, d->lddh, d->kept, d->act, d->M, F, dz, lddz, pg, pu, stream));
    if (pg != nullptr || pu != nullptr) TO_TRY(tok_column_sums(pg, pu, to_nblk(d->M), F, d->dbg, d->dbu, stream));
    TgOperand W{d->wg, d->wu, d->ldw, false}, X{d->x, d->x, d->ldx, false};
    ToCopies copies;
    if (w.pack_w) {
        W = copies.add(d->wg, d->ldw, F, d->K, ws + w.w);
        W.p2 = copies.add(d->wu, d->ldw, F, d->K, ws + w.w + tok_align((size_t)F * to_pitch(d->K) * es)).p;
    }
    if (w.pack_x) X = copies.add(d->x, d->ldx, d->M, d->K, ws + w.x);
    TO_TRY(copies.go(d->dtype, stream));
    TgSum sx{}, sw{};
    if (d->dx != nullptr) {
        TgArgs a{};
        a.ranges = a.batches = 1;
        a.a = TgOperand{dz, du, lddz, true};
        a.b = W;
        a.M = d->M; a.N = d->K; a.K = F;
        a.ranges = 2;
        a.y = a.y2 = d->dx; a.ldy = d->lddx;
        TO_TRY(tg_launch(d->dtype, 0, 1, TG_STORE, a, (float*)(ws + w.slab_x), stream, &sx));
    }
    if (d->dwg != nullptr) {
        TgArgs a{};
        a.ranges = a.batches = 1;
        a.a = TgOperand{dz, du, lddz, true};
        a.b = X;
        a.M = F; a.N = d->K; a.K = d->M;
        a.y = d->dwg; a.y2 = d->dwu; a.ldy = d->lddw; a.batches = 2;
        TO_TRY(tg_launch(d->dtype, 1, 1, TG_STORE, a, (float*)(ws + w.slab_w), stream, &sw));
    }
    return tg_sums(d->dtype, sx, sw, stream);
}
