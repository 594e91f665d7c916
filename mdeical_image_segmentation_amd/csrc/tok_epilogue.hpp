// Epilogues of the token products: a lane holds runs of 8 consecutive columns of one row.  ACT: the activation, or -1: the descriptor's (a kernel that unrolls many rows takes it as a
// template argument - six activations in each row make the code too long to unroll).
#pragma once
#include "tok_gemm.hpp"

// where batch bt is stored (p + s (p2 - p), not s ? p2 : p: hipcc turns that into an indexed load from a scratch copy of the arguments)
__device__ __forceinline__ char* tg_out(const TgArgs& a, int bt) { return (char*)a.y + (long long)bt * ((char*)a.y2 - (char*)a.y); }

// y = act(v + bias) + res
template <typename T, int ACT = -1> struct TgLinearRow {
    const TgArgs& a;
    long long n;            // first column of the run
    int nv;                 // columns of it inside the matrix
    void* y;
    float bias[8];
    __device__ __forceinline__ TgLinearRow(const TgArgs& a_, void* y_, long long n_, bool full) : a(a_), n(n_), nv(a_.N - n_ >= 8 ? 8 : (int)(a_.N - n_)), y(y_) {
        if (full && a.bias != nullptr && nv > 0) tok_ldn<float>(a.bias + n, bias, nv);
    }
    __device__ __forceinline__ void store(long long m, const float (&v)[8]) const { tok_stn<T>(reinterpret_cast<T*>(y) + m * a.ldy + n, v, nv); }
    __device__ __forceinline__ void operator()(long long m, float (&v)[8]) const {
        if (a.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += bias[j];
        }
        if (a.kept != nullptr) tok_stn<float>(a.kept + m * a.N + n, v, nv);
        tok_act8<sizeof(T) == 4, false>(ACT < 0 ? a.act : ACT, v, nullptr);
        if (a.res != nullptr) {
            float r[8];
            tok_ldn<T>(reinterpret_cast<const T*>(a.res) + m * a.ldres + n, r, nv);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += r[j];
        }
        store(m, v);
    }
};
// h = act(g + bg) (u + bu)
template <typename T, int ACT = -1> struct TgGatedRow {
    const TgArgs& a;
    long long n;
    int nv;
    float bg[8], bu[8];
    __device__ __forceinline__ TgGatedRow(const TgArgs& a_, long long n_) : a(a_), n(n_), nv(a_.N - n_ >= 8 ? 8 : (int)(a_.N - n_)) {
        if (a.bias != nullptr && nv > 0) tok_ldn<float>(a.bias + n, bg, nv);
        if (a.bias2 != nullptr && nv > 0) tok_ldn<float>(a.bias2 + n, bu, nv);
    }
    __device__ __forceinline__ void operator()(long long m, float (&g)[8], float (&u)[8]) const {
        if (a.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] += bg[j];
        }
        if (a.bias2 != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] += bu[j];
        }
        if (a.kept != nullptr) {
            tok_stn<float>(a.kept + m * a.N + n, g, nv);
            tok_stn<float>(a.kept2 + m * a.N + n, u, nv);
        }
        tok_act8<sizeof(T) == 4, false>(ACT < 0 ? a.act : ACT, g, nullptr);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] *= u[j];
        tok_stn<T>(reinterpret_cast<T*>(a.y) + m * a.ldy + n, g, nv);
    }
};
