// layer_norm_kernel.hpp -- layer norm over the last axis, forward and backward
// (gfx950).
//
//   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   xh = (x - mean) rstd, g = dy w:  dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Both directions are bound by HBM: a row is read once into registers, its
// statistics are sums over the team of lanes that holds it, and the result is
// written from the registers.  The mean is taken twice, as the sum's and as the
// mean of the distances from that, which a row's size no longer rounds: a row of one
// value v has mean v and variance 0 (from the sum alone 15 values of 1e4 came out at
// -0.3).  The squared distances from it follow.  The third sum costs nothing where HBM bounds, and 0.2 us on a single
// row.  2.4M rows of 128 fp32 values: forward 449 us (5.6 TB/s), backward 665 us
// (5.7 TB/s) and 5 us to join the partial sums of dw and db; 8192 rows of 4096 bf16
// values forward 25 us (5.4 TB/s).  A copy of 1 GiB reaches 5.1 TB/s.
//
// FMAs are written out and others forbidden, so the rows' bits do not depend on
// which variant of a kernel takes them, that is on how many rows there are.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "train_common.hpp"

namespace tca {

struct LayerNormArgs {
    const void* x;   // rows x n, pitch elements apart
    const void* w;   // NULL: ones
    const void* b;   // NULL: zeros
    void* y;         // rows x n, dense
    float2* stats;   // [rows] {mean, rstd}, or NULL
    int64_t rows, pitch;
    int n;
    float eps, inv_n;
    bool w_f32;
    int w_half;      // w's 16-bit type is XT (0) or YT (1)
};

// A weight vector (w or b) as fp32: `fill` if there is none.
template <typename XT, typename YT, int E>
__device__ __forceinline__ void norm_weight(const void* p, bool f32, int half, int at, float fill, float (&out)[E]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = fill;
    } else if (half == 0) {
        load_weight<XT, E>(p, f32, at, out);
    } else {
        load_weight<YT, E>(p, f32, at, out);
    }
}

// A team takes R rows a turn: their loads are in flight together and their sums
// share steps and barriers.
template <typename XT, typename YT, int E, int G, int V, int R, bool kStream>
__global__ __launch_bounds__(team_threads(G)) void layer_norm_kernel(LayerNormArgs a) {
#pragma clang fp contract(off)
    constexpr int kTeams = team_threads(G) / G;
    __shared__ float lds[G > 64 ? 2 * R * G / 64 : 1];
    Team<G, R, Add> sum(lds);
    const int lane = threadIdx.x % G;
    const Columns<E, G, V> col(lane, a.n);
    float w[V][E], b[V][E];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        norm_weight<XT, YT, E>(a.w, a.w_f32, a.w_half, col.at[v], 1.0f, w[v]);
        norm_weight<XT, YT, E>(a.b, a.w_f32, a.w_half, col.at[v], 0.0f, b[v]);
    }
    // every team of a workgroup runs as many turns as its first one: the lanes of a
    // wavefront stay together in the sums
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * kTeams * R; first < a.rows;
         first += static_cast<int64_t>(gridDim.x) * kTeams * R) {
        const int64_t row = first + threadIdx.x / G;  // and every kTeams-th after it
        Pack<XT, E> raw[R][V];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const XT* x = static_cast<const XT*>(a.x) + min(row + r * kTeams, a.rows - 1) * a.pitch;
#pragma unroll
            for (int v = 0; v < V; ++v) raw[r][v] = load_any<XT, E, kStream>(x + col.at[v]);
        }
        float mean[R], s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) mean[r] = 0.0f;
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {  // the sum's mean, then what it is off by
#pragma unroll
            for (int r = 0; r < R; ++r) {
                s[r] = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int i = 0; i < E; ++i) s[r] += col.counts(v, i) ? to_f32(raw[r][v].v[i]) - mean[r] : 0.0f;
            }
            sum(s);
#pragma unroll
            for (int r = 0; r < R; ++r) mean[r] += s[r] * a.inv_n;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[r] = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float d = to_f32(raw[r][v].v[i]) - mean[r];
                    s[r] = col.counts(v, i) ? __builtin_fmaf(d, d, s[r]) : s[r];
                }
        }
        sum(s);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t at = row + r * kTeams;
            const float rstd = 1.0f / sqrtf(__builtin_fmaf(s[r], a.inv_n, a.eps));
            if (at >= a.rows) break;
            YT* y = static_cast<YT*>(a.y) + at * a.n;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float out[E];
#pragma unroll
                for (int i = 0; i < E; ++i) out[i] = __builtin_fmaf((to_f32(raw[r][v].v[i]) - mean[r]) * rstd, w[v][i], b[v][i]);
                if (col.inside(v)) store_any<YT, E, kStream>(y + col.at[v], round_pack<YT, E>(out));
            }
            if (a.stats && lane == 0) a.stats[at] = make_float2(mean[r], rstd);
        }
    }
}

struct LayerNormBackArgs {
    const void* dy;  // rows x n, dy_pitch elements apart
    const void* x;
    const void* w;
    const float2* stats;
    void* dx;        // dense, or NULL
    float* partial;  // [workgroups][2][n]: the rows' sums of dy xh and of dy
    int64_t rows, pitch, dy_pitch;
    int n;
    float inv_n;
    bool w_f32;
    int w_half;
};

// dx, and the sums over this workgroup's rows that dw and db are made of.
template <typename XT, typename YT, int E, int G, int V, int R, bool kStream>
__global__ __launch_bounds__(team_threads(G)) void layer_norm_back_kernel(LayerNormBackArgs a) {
#pragma clang fp contract(off)
    constexpr int kTeams = team_threads(G) / G;
    constexpr int kWidth = G * V * E;
    __shared__ float lds[G > 64 ? 4 * R * G / 64 : 1];
    __shared__ float joined[kTeams > 1 ? kTeams * kWidth : 1];
    Team<G, 2 * R, Add> sum(lds);
    const int lane = threadIdx.x % G;
    const Columns<E, G, V> col(lane, a.n);
    float w[V][E], dw[V][E] = {}, db[V][E] = {};
#pragma unroll
    for (int v = 0; v < V; ++v) norm_weight<XT, YT, E>(a.w, a.w_f32, a.w_half, col.at[v], 1.0f, w[v]);
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * kTeams * R; first < a.rows;
         first += static_cast<int64_t>(gridDim.x) * kTeams * R) {
        const int64_t row = first + threadIdx.x / G;
        Pack<XT, E> rx[R][V];
        Pack<YT, E> rg[R][V];
        float2 st[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t from = min(row + r * kTeams, a.rows - 1);
            const XT* x = static_cast<const XT*>(a.x) + from * a.pitch;
            const YT* dy = static_cast<const YT*>(a.dy) + from * a.dy_pitch;
            st[r] = a.stats[from];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                rx[r][v] = load_any<XT, E, kStream>(x + col.at[v]);
                rg[r][v] = load_any<YT, E, kStream>(dy + col.at[v]);
            }
        }
        float s[2 * R] = {};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool mine = row + r * kTeams < a.rows;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float xh = (to_f32(rx[r][v].v[i]) - st[r].x) * st[r].y;
                    const float d = to_f32(rg[r][v].v[i]);
                    const float g = d * w[v][i];
                    if (col.counts(v, i)) {
                        s[2 * r] += g;
                        s[2 * r + 1] = __builtin_fmaf(g, xh, s[2 * r + 1]);
                        if (mine) {
                            dw[v][i] = __builtin_fmaf(d, xh, dw[v][i]);
                            db[v][i] += d;
                        }
                    }
                }
        }
        if (!a.dx) continue;
        sum(s);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t at = row + r * kTeams;
            if (at >= a.rows) break;
            const float mg = s[2 * r] * a.inv_n, mgx = s[2 * r + 1] * a.inv_n;
            XT* dx = static_cast<XT*>(a.dx) + at * a.n;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float out[E];
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float xh = (to_f32(rx[r][v].v[i]) - st[r].x) * st[r].y;
                    out[i] = st[r].y * __builtin_fmaf(-xh, mgx, __builtin_fmaf(to_f32(rg[r][v].v[i]), w[v][i], -mg));
                }
                if (col.inside(v)) store_any<XT, E, kStream>(dx + col.at[v], round_pack<XT, E>(out));
            }
        }
    }
    if (!a.partial) return;
    float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.n;
#pragma unroll
    for (int half = 0; half < 2; ++half, out += a.n) {
        if constexpr (kTeams == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (col.counts(v, i)) out[col.at[v] + i] = half ? db[v][i] : dw[v][i];
        } else {
            if (half) __syncthreads();
            float* mine = joined + threadIdx.x / G * kWidth;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (col.counts(v, i)) mine[col.at[v] + i] = half ? db[v][i] : dw[v][i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.n; c += team_threads(G)) {
                float s = 0.0f;
#pragma unroll
                for (int t = 0; t < kTeams; ++t) s += joined[t * kWidth + c];
                out[c] = s;
            }
        }
    }
}

// The columns' sums over the workgroups' partial rows, rounded into dw (columns
// [0, n) of a partial row) and db (the rest).  A workgroup takes 32 columns in
// lanes of 4; its kSlots slots split the partial rows and meet in LDS; orders are
// fixed.
constexpr int kNormJoinCols = 32, kNormJoinSlots = 128;
template <typename WT>
__global__ __launch_bounds__(8 * kNormJoinSlots) void layer_norm_join_kernel(const float* partial, int parts, int n,
                                                                             WT* dw, WT* db) {
    __shared__ float lds[kNormJoinSlots][kNormJoinCols + 1];
    const int slot = threadIdx.x / 8, at = threadIdx.x % 8 * 4;
    const int width = 2 * n, col = blockIdx.x * kNormJoinCols + at;
    float s[4] = {};
    if (col + 4 <= width) {
#pragma unroll 4
        for (int p = slot; p < parts; p += kNormJoinSlots) {
            const auto v = load_any<float, 4>(partial + static_cast<int64_t>(p) * width + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += v.v[i];
        }
    } else {
        for (int p = slot; p < parts; p += kNormJoinSlots)
            for (int i = 0; col + i < width; ++i) s[i] += partial[static_cast<int64_t>(p) * width + col + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[slot][at + i] = s[i];
    __syncthreads();
    // 32 lanes per column, 4 slots each
    const int c = threadIdx.x / 32, part = threadIdx.x % 32;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < kNormJoinSlots / 32; ++k) t += lds[k * 32 + part][c];
    t = team_combine<32>(t, Add());
    const int out_col = blockIdx.x * kNormJoinCols + c;
    if (part == 0 && out_col < width) {
        WT* out = out_col < n ? dw : db;
        if (out) out[out_col < n ? out_col : out_col - n] = from_f32<WT>(t);
    }
}

}  // namespace tca
