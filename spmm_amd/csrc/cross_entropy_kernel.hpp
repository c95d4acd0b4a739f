// cross_entropy_kernel.hpp -- softmax cross entropy and its gradient (gfx950).
//
//   m = max_c x, s = sum_c exp(x - m);  loss = log(s) - (x_t - m)
//   dx = (exp(x - m) / s - [c = t]) * scale
//
// m and s are kept apart (not as m + log(s)): exp(x - m) / s has the precision
// of its parts however large the logits are.  All of it is bound by HBM: a row
// is read once into registers, its maximum and its sum are taken over the team
// of lanes that holds it, and the gradient is written from the registers
// (exp is computed twice rather than kept: the registers hold the row in its
// own type).  Rows without a label are not read.  No operations are contracted
// into FMAs, so a row's bits do not depend on the variant that takes it.
//
// 4096 x 50001 bf16 logits, three quarters with a label, loss and gradient at once
// 160 us (4.5 TB/s; 143 us, 5.0 TB/s, at 50048 classes, whose rows start on whole
// lines); 2048 x 32768 fp32 forward 48 us (5.6 TB/s), backward 77 us; 2.4M rows of
// 47 fp32 logits, 8 % with a label, forward 36 us, backward 118 us (590 MB through
// HBM, 5.0 TB/s).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "train_common.hpp"

namespace tca {

constexpr int kLossParts = 256;  // workgroups that count rows

enum LossMode { kLossForward, kLossBackward, kLossBoth };

struct CrossEntropyArgs {
    const void* x;          // rows x n, pitch elements apart
    const void* targets;
    void* dx;               // rows x n, dense
    float* row_loss;        // [rows], or NULL
    float2* stats;          // [rows] {m, s}: written forward (unless NULL), read backward
    float2* parts;          // [workgroups] {loss, count's bits}, or NULL
    const int* counts;      // kLossBoth: [kLossParts] rows that count, or NULL (sum)
    const float* gloss;     // kLossBackward
    const float* norm;      // kLossBackward, or NULL (1)
    int64_t gloss_stride, ignore;
    int rows, n, pitch;
    float scale;            // kLossBoth
    bool wide_targets;      // int64
    bool own_count;         // kLossBoth: the mean's count is each workgroup's own work
};

__device__ __forceinline__ int64_t load_target(const CrossEntropyArgs& a, int64_t row) {
    return a.wide_targets ? static_cast<const int64_t*>(a.targets)[row]
                          : static_cast<int64_t>(static_cast<const int*>(a.targets)[row]);
}

// exp(d): the hardware's exp2 of d log2(e).  The product's rounding is relative to
// |d|, and so is the result's error, |d| 2^-24: largest where exp(d), d <= 0, is
// smallest.  Results below 2^-126 are 0.
// (One FMA, x log2(e) - m log2(e), saves an instruction and overflows for logits
// near fp32's ends, which masks use.)
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }

// Rows with a label among every `step`-th from `first` on, four loads in flight.
__device__ __forceinline__ int count_labels(const CrossEntropyArgs& a, int64_t first, int64_t step) {
    int n = 0;
    for (int64_t row = first; row < a.rows; row += 4 * step) {
        int64_t t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = row + k * step < a.rows ? load_target(a, row + k * step) : a.ignore;
#pragma unroll
        for (int k = 0; k < 4; ++k) n += t[k] != a.ignore;
    }
    return n;
}

// Rows that count, over all of them: what the mean divides by.
constexpr int kLossCountThreads = 1024;
__global__ __launch_bounds__(kLossCountThreads) void loss_count_kernel(CrossEntropyArgs a, int* counts) {
    __shared__ int lds[kLossCountThreads / 64];
    int n = count_labels(a, static_cast<int64_t>(blockIdx.x) * kLossCountThreads + threadIdx.x,
                         static_cast<int64_t>(gridDim.x) * kLossCountThreads);
    for (int step = 32; step; step >>= 1) n += __shfl_xor(n, step);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLossCountThreads / 64; ++w) n += lds[w];
        counts[blockIdx.x] = n;
    }
}

// What a workgroup's rows add to the loss, from lane values of its teams.
template <int kThreads>
__device__ __forceinline__ void store_part(const CrossEntropyArgs& a, float loss, int count) {
    __shared__ float lds_loss[kThreads / 64];
    __shared__ int lds_count[kThreads / 64];
    loss = team_combine<64>(loss, Add());
    for (int step = 32; step; step >>= 1) count += __shfl_xor(count, step);
    if ((threadIdx.x & 63) == 0) {
        lds_loss[threadIdx.x >> 6] = loss;
        lds_count[threadIdx.x >> 6] = count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 64; ++w) {
            loss += lds_loss[w];
            count += lds_count[w];
        }
        a.parts[blockIdx.x] = make_float2(loss, __int_as_float(count));
    }
}

// 1 / count of the mean (0 over no rows: every gradient is 0 then): from
// loss_count_kernel's parts, or each wavefront counts; the same in every lane.
__device__ __forceinline__ float mean_factor(const CrossEntropyArgs& a) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    if (a.own_count) {
        n = count_labels(a, lane, 64);
    } else {
        for (int k = 0; k < kLossParts / 64; ++k) n += a.counts[k * 64 + lane];
    }
    for (int step = 32; step; step >>= 1) n += __shfl_xor(n, step);
    return n ? 1.0f / static_cast<float>(n) : 0.0f;
}

// The larger of t and E values.
template <typename T, int E>
__device__ __forceinline__ float max_of(const Pack<T, E>& v, float t) {
#pragma unroll
    for (int i = 0; i + 1 < E; i += 2) {
        const float a = to_f32(v.v[i]), b = to_f32(v.v[i + 1]);
        float r;
        asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(t));  // fmaxf would quiet each operand first
        t = r;
    }
    if constexpr (E % 2) t = fmaxf(t, to_f32(v.v[E - 1]));
    return t;
}

// What a row brings with it: its place, its target, and per mode its statistics.
struct LossRow {
    int offset;    // from the chunk's first row
    int target;    // a class, kNoLabel or kBadLabel
    float xt;      // the target's logit (forward)
    float2 stats;  // backward
    float scale;   // backward
};
constexpr int kNoLabel = -1, kBadLabel = -2;

// G lanes take a row, V vectors of E each.  A unit -- a wavefront, or the
// workgroup where a row takes more -- walks chunks of `chunk` rows (at most 64): it
// reads their targets in one access, the next chunk's while this one is worked
// on, and takes S * R rows a turn; where a gradient is written and rows are narrow,
// those of the next turn are in flight during this one (elsewhere the registers
// are better spent on more wavefronts: 4096 x 50001 bf16 logits 159 us, 177 with the
// next row in flight; a million rows of 100 fp16 logits forward 58 and 64).
// Forward, only the rows with a label are walked; so they are for a gradient of
// narrow rows (a chunk's lie in one piece) of which a quarter or more have no label,
// once the chunk is cleared in whole accesses.
template <typename T, int kMode, int E, int G, int V, int R, bool kStream>
__global__ __launch_bounds__(team_threads(G)) void cross_entropy_kernel(CrossEntropyArgs a, int chunk) {
#pragma clang fp contract(off)
    constexpr int S = G < 64 ? 64 / G : 1;
    constexpr int kUnits = G > 64 ? 1 : team_threads(G) / 64;
    constexpr bool kAhead = G <= 64 && V <= 2 && kMode != kLossForward;
    __shared__ float lds_max[G > 64 ? 2 * R * G / 64 : 1], lds_sum[G > 64 ? 2 * R * G / 64 : 1];
    Team<G, R, Max> max(lds_max);
    Team<G, R, Add> sum(lds_sum);
    const int lane = threadIdx.x % G, wave_lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Columns<E, G, V> col(lane, a.n);
    float total = 0.0f;
    int count = 0;
    float scale = 0.0f;
    if constexpr (kMode == kLossBoth) scale = a.counts || a.own_count ? a.scale * mean_factor(a) : a.scale;
    if constexpr (kMode == kLossBackward) {
        scale = a.norm ? *a.norm : 1.0f;
        if (a.gloss_stride == 0) scale *= *a.gloss;
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * kUnits * chunk;
    int64_t base = (static_cast<int64_t>(blockIdx.x) * kUnits + (G > 64 ? 0 : wave)) * chunk;
    const auto chunk_target = [&](int64_t at) {
        return wave_lane < chunk && at + wave_lane < a.rows ? load_target(a, at + wave_lane) : a.ignore;
    };
    int64_t next_target = chunk_target(base);
    for (; base < a.rows; base += step) {
        const int64_t target = next_target;
        next_target = chunk_target(base + step);
        const int here = static_cast<int>(min(static_cast<int64_t>(chunk), a.rows - base));
        const bool labelled = target != a.ignore;
        const int label = !labelled ? kNoLabel : target < 0 || target >= a.n ? kBadLabel : static_cast<int>(target);
        const uint64_t mask = __ballot(labelled);
        const int labels = __popcll(mask);
        const bool clear = kMode != kLossForward && G <= 64 && labels * 4 <= here * 3;
        int items = here, order = wave_lane;
        if (kMode == kLossForward || clear) {  // rows with a label first
            items = labels;
            const int before = __popcll(mask & ((1ull << wave_lane) - 1));
            order = __builtin_amdgcn_ds_permute(4 * (labelled ? before : items + wave_lane - before), wave_lane);
        }
        if (kMode == kLossForward && a.row_loss && wave_lane < here && !labelled && (G <= 64 || wave == 0))
            a.row_loss[base + wave_lane] = 0.0f;
        if (wave_lane == 0 && (G <= 64 || wave == 0)) count += labels;
        T* const dx0 = kMode == kLossForward ? nullptr : static_cast<T*>(a.dx) + base * a.n;
        const T* const x0 = static_cast<const T*>(a.x) + base * static_cast<int64_t>(a.pitch);
        const auto fetch = [&](int first, LossRow (&row)[R], Pack<T, E> (&raw)[R][V]) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int item = first + r * S + (G < 64 ? wave_lane / G : 0);
                const int from = item < items ? item : 0;
                if constexpr (S == 1) {
                    row[r].offset = __builtin_amdgcn_readlane(order, from);
                    row[r].target = __builtin_amdgcn_readlane(label, row[r].offset);
                } else {
                    row[r].offset = __shfl(order, from);
                    row[r].target = __shfl(label, row[r].offset);
                }
                if (item >= items) row[r].target = kNoLabel;
                if (row[r].target != kNoLabel) {
                    const T* const x = x0 + static_cast<int64_t>(row[r].offset) * a.pitch;
#pragma unroll
                    for (int v = 0; v < V; ++v) raw[r][v] = load_any<T, E, kStream>(x + col.at[v]);
                    if constexpr (kMode == kLossBackward) {
                        row[r].stats = a.stats[base + row[r].offset];
                        row[r].scale = a.gloss_stride ? a.gloss[(base + row[r].offset) * a.gloss_stride] * scale : scale;
                    } else {
                        row[r].xt = row[r].target >= 0 ? to_f32(x[row[r].target]) : 0.0f;
                    }
                }
            }
        };
        LossRow row[R];
        Pack<T, E> raw[R][V] = {};
        fetch(0, row, raw);  // in flight while the chunk is cleared
        if constexpr (kMode != kLossForward && G <= 64) {
            if (clear) {
                constexpr int Z = 16 / sizeof(T);
                const int values = here * a.n;  // at most 64 rows of 384 vectors
                for (int c = wave_lane * Z; c < values; c += 64 * Z) {
                    if (c + Z <= values) {
                        store_any<T, Z>(dx0 + c, Pack<T, Z>{});
                    } else {
                        for (int i = c; i < values; ++i) dx0[i] = T{};
                    }
                }
                // the rows with a label are written over it: by other lanes, after it
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
        }
        for (int first = 0; first < items; first += S * R) {
            LossRow next_row[R];
            Pack<T, E> next_raw[R][V] = {};
            if (kAhead && first + S * R < items) fetch(first + S * R, next_row, next_raw);
            float top[R], s[R];
            if constexpr (kMode == kLossBackward) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    top[r] = row[r].stats.x;
                    s[r] = row[r].stats.y;
                }
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float t = -__builtin_inff();
#pragma unroll
                    for (int v = 0; v < V; ++v) t = max_of(raw[r][v], t);  // twice-read values included
                    top[r] = fmaxf(t, t);
                }
                max(top);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    s[r] = 0.0f;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        forget(raw[r][v]);
#pragma unroll
                        for (int i = 0; i < E; ++i) {
                            const float term = exp_of(to_f32(raw[r][v].v[i]) - top[r]);
                            s[r] += v < V - 1 ? term : col.counts(v, i) ? term : 0.0f;
                        }
                    }
                }
                sum(s);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int item = first + r * S + (G < 64 ? wave_lane / G : 0);
                const int64_t at = base + row[r].offset;
                const int target = row[r].target;
                if constexpr (kMode != kLossBackward) {
                    if (lane == 0 && target != kNoLabel) {
                        const float loss = target == kBadLabel ? __builtin_nanf("") : logf(s[r]) - (row[r].xt - top[r]);
                        if (a.stats) a.stats[at] = make_float2(top[r], s[r]);
                        if (a.row_loss) a.row_loss[at] = loss;
                        total += loss;
                    }
                }
                if constexpr (kMode != kLossForward) {
                    if (item < items) {
                        T* const dx = dx0 + (G <= 64 ? row[r].offset * a.n : static_cast<int64_t>(row[r].offset) * a.n);
                        float k = kMode == kLossBackward ? row[r].scale : scale;
                        if (target == kBadLabel) k = __builtin_nanf("");
                        const float factor = k / s[r];
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            float out[E];
                            forget(raw[r][v]);
                            if (target != kNoLabel) {
#pragma unroll
                                for (int i = 0; i < E; ++i) out[i] = exp_of(to_f32(raw[r][v].v[i]) - top[r]) * factor;
                                const unsigned hit = static_cast<unsigned>(target - col.at[v]);
                                if (hit < E) {
#pragma unroll
                                    for (unsigned i = 0; i < E; ++i) out[i] -= hit == i ? k : 0.0f;
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < E; ++i) out[i] = 0.0f;
                            }
                            if (col.inside(v)) store_any<T, E, kStream>(dx + col.at[v], round_pack<T, E>(out));
                        }
                    }
                }
            }
            if constexpr (kAhead) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    row[r] = next_row[r];
#pragma unroll
                    for (int v = 0; v < V; ++v) raw[r][v] = next_raw[r][v];
                }
            } else if (first + S * R < items) {
                fetch(first + S * R, row, raw);
            }
        }
    }
    if constexpr (kMode != kLossBackward) {
        if (a.parts) store_part<team_threads(G)>(a, total, count);
    }
}

// Rows of more than 1024 vectors, of any length: a workgroup walks a row in steps
// of kLongVecs vectors per lane.  Forward and backward read it once: forward, each
// lane keeps a running maximum and the sum under it, scaled down when a step brings
// a larger one.  Both at once read it twice, and take rows that the registers hold
// no more (cross_entropy_kernel has the others).
constexpr int kLongThreads = 512, kLongVecs = 4;

// fn(first column, vectors) over a row's whole vectors: kLongVecs at a time, then
// one by one; the columns after the last whole vector are left.
template <int E, typename F>
__device__ __forceinline__ void long_walk(int n, F&& fn) {
    constexpr int kStep = kLongThreads * E;
    int c = 0;
    for (; c + kLongVecs * kStep <= n; c += kLongVecs * kStep)
        fn(c + static_cast<int>(threadIdx.x) * E, std::integral_constant<int, kLongVecs>());
    for (c += static_cast<int>(threadIdx.x) * E; c + E <= n; c += kStep) fn(c, std::integral_constant<int, 1>());
}

template <typename T, int kMode, bool kStream>
__global__ __launch_bounds__(kLongThreads) void cross_entropy_long_kernel(CrossEntropyArgs a) {
#pragma clang fp contract(off)
    constexpr int E = 16 / sizeof(T), kStep = kLongThreads * E;
    __shared__ float lds_max[2 * kLongThreads / 64], lds_sum[2 * kLongThreads / 64];
    Team<kLongThreads, 1, Max> max(lds_max);
    Team<kLongThreads, 1, Add> sum(lds_sum);
    float total = 0.0f;
    int count = 0;
    float scale = 0.0f;
    if constexpr (kMode == kLossBoth) scale = a.counts || a.own_count ? a.scale * mean_factor(a) : a.scale;
    const int tail = a.n / E * E + threadIdx.x;  // this lane's column after the last whole vector, if it is in the row
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t target = load_target(a, row);
        const bool labelled = target != a.ignore;
        const bool bad = labelled && (target < 0 || target >= a.n);
        const T* x = static_cast<const T*>(a.x) + row * static_cast<int64_t>(a.pitch);
        float top = 0.0f, s = 1.0f;
        if constexpr (kMode == kLossBackward) {
            if (labelled) {
                const float2 st = a.stats[row];
                top = st.x;
                s = st.y;
                scale = a.gloss[row * a.gloss_stride] * (a.norm ? *a.norm : 1.0f);
            }
        } else if (labelled) {
            const float xt = bad ? 0.0f : to_f32(x[target]);
            float m = -__builtin_inff(), l = 0.0f;  // the sum of exp(x - m); 0 under m = -inf
            const auto grow = [&](float big) {
                const float old = m;
                m = fmaxf(m, big);
                const float under = m == -__builtin_inff() ? 0.0f : m;  // exp(-inf - under) = 0
                l *= exp_of(old - under);
                return under;
            };
            long_walk<E>(a.n, [&](int c, auto many) {
                constexpr int V = decltype(many)::value;
                Pack<T, E> raw[V];
#pragma unroll
                for (int v = 0; v < V; ++v) raw[v] = load_any<T, E, kStream && kMode == kLossForward>(x + c + v * kStep);
                float big = -__builtin_inff();
#pragma unroll
                for (int v = 0; v < V; ++v) big = max_of(raw[v], big);
                const float under = grow(big);
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int i = 0; i < E; ++i) l += exp_of(to_f32(raw[v].v[i]) - under);
            });
            if (tail < a.n) {
                const float v = to_f32(x[tail]);
                l += exp_of(v - grow(v));
            }
            float t[1] = {m};
            max(t);
            top = t[0];
            t[0] = m == -__builtin_inff() ? l : l * exp_of(m - top);  // nothing but -inf: l is 0, or NaN
            sum(t);
            s = top == -__builtin_inff() ? __builtin_nanf("") : t[0];
            if (threadIdx.x == 0) {
                const float loss = bad ? __builtin_nanf("") : logf(s) - (xt - top);
                if (a.stats) a.stats[row] = make_float2(top, s);
                if (a.row_loss) a.row_loss[row] = loss;
                total += loss;
                count += 1;
            }
        } else if (a.row_loss && threadIdx.x == 0) {
            a.row_loss[row] = 0.0f;
        }
        if constexpr (kMode != kLossForward) {
            T* dx = static_cast<T*>(a.dx) + row * a.n;
            const float k = bad ? __builtin_nanf("") : scale, factor = k / s;
            const int hit = labelled && !bad ? static_cast<int>(target) : -1;
            long_walk<E>(a.n, [&](int c, auto many) {
                constexpr int V = decltype(many)::value;
                Pack<T, E> raw[V] = {};
                if (labelled) {
#pragma unroll
                    for (int v = 0; v < V; ++v) raw[v] = load_any<T, E, kStream>(x + c + v * kStep);
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float out[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) out[i] = labelled ? exp_of(to_f32(raw[v].v[i]) - top) * factor : 0.0f;
                    const unsigned at = static_cast<unsigned>(hit - (c + v * kStep));
                    if (hit >= 0 && at < E) {
#pragma unroll
                        for (unsigned i = 0; i < E; ++i) out[i] -= at == i ? k : 0.0f;
                    }
                    store_any<T, E, kStream>(dx + c + v * kStep, round_pack<T, E>(out));
                }
            });
            if (tail < a.n) {
                const float p = labelled ? exp_of(to_f32(x[tail]) - top) * factor : 0.0f;
                dx[tail] = from_f32<T>(tail == hit ? p - k : p);
            }
        }
    }
    if constexpr (kMode != kLossBackward) {
        if (a.parts) store_part<kLongThreads>(a, total, count);
    }
}

// The workgroups' parts joined (in fp64, in a fixed order): the loss, and the
// factor of the mean for the backward pass.
constexpr int kLossJoinThreads = 512;
__global__ __launch_bounds__(kLossJoinThreads) void loss_join_kernel(const float2* parts, int n, bool mean, float* loss,
                                                                     float* norm) {
    constexpr int W = kLossJoinThreads / 64;
    __shared__ double lds[W];
    __shared__ int64_t lds_count[W];
    double total = 0.0;
    int64_t count = 0;
#pragma unroll 4
    for (int k = threadIdx.x; k < n; k += kLossJoinThreads) {
        total += parts[k].x;
        count += __float_as_int(parts[k].y);
    }
    for (int step = 32; step; step >>= 1) {
        total += __shfl_xor(total, step);
        count += __shfl_xor(count, step);
    }
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = total;
        lds_count[threadIdx.x >> 6] = count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < W; ++w) {
            total += lds[w];
            count += lds_count[w];
        }
        if (loss) *loss = static_cast<float>(mean && count ? total / static_cast<double>(count) : total);
        if (norm) *norm = mean ? (count ? 1.0f / static_cast<float>(count) : 0.0f) : 1.0f;
    }
}

}  // namespace tca
