// train_common.hpp -- what the training operators' kernels share: vectors of
// any element alignment, sums and maxima over teams of lanes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "value_types.hpp"

namespace tca {

// The unsigned vector of `bytes` bytes that one access moves, at any address.
template <int kBytes>
struct Word {
    typedef uint32_t plain __attribute__((ext_vector_type(kBytes / 4)));
    typedef plain type __attribute__((aligned(1)));
};
template <>
struct Word<4> {
    typedef uint32_t plain;
    typedef plain type __attribute__((aligned(1)));
};
template <>
struct Word<2> {
    typedef uint16_t plain;
    typedef plain type __attribute__((aligned(1)));
};

// E values at p, which needs its element's alignment only: one global access
// (the hardware takes 16-byte accesses at any address).  kStream: with the
// caches told that the line is used once, for passes over more than they hold.
template <typename T, int E, bool kStream = false>
__device__ __forceinline__ Pack<T, E> load_any(const T* p) {
    using W = Word<sizeof(Pack<T, E>)>;
    const auto* w = reinterpret_cast<const typename W::type*>(p);
    typename W::plain v;
    if constexpr (kStream) v = __builtin_nontemporal_load(w);
    else v = *w;
    return __builtin_bit_cast(Pack<T, E>, v);
}

template <typename T, int E, bool kStream = false>
__device__ __forceinline__ void store_any(T* p, const Pack<T, E>& x) {
    using W = Word<sizeof(Pack<T, E>)>;
    auto* w = reinterpret_cast<typename W::type*>(p);
    const auto v = __builtin_bit_cast(typename W::plain, x);
    if constexpr (kStream) __builtin_nontemporal_store(v, w);
    else *w = v;
}

template <typename T>
__device__ __forceinline__ T from_f32(float x) {
    if constexpr (sizeof(T) == 4) {
        return x;
    } else if constexpr (__is_same(T, _Float16)) {
        // x is an fp32 value first: without this the compiler turns some FMAs and their
        // conversion into one instruction that rounds once, in some places of a kernel
        // and not in others, and a row's bits depend on its place among the rows
        asm("" : "+v"(x));
        return static_cast<_Float16>(x);
    } else {
        return __builtin_bit_cast(bf16_t, static_cast<__bf16>(x));  // v_cvt_pk_bf16_f32: nearest even
    }
}

template <typename T, int E>
__device__ __forceinline__ Pack<T, E> round_pack(const float (&x)[E]) {
    Pack<T, E> r;
#pragma unroll
    for (int i = 0; i < E; ++i) r.v[i] = from_f32<T>(x[i]);
    return r;
}

// E values of `p` (fp32 if f32, else T) as fp32.
template <typename T, int E>
__device__ __forceinline__ void load_weight(const void* p, bool f32, int64_t at, float (&out)[E]) {
    if (f32) {
        const auto v = load_any<float, E>(static_cast<const float*>(p) + at);
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = v.v[i];
    } else {
        const auto v = load_any<T, E>(static_cast<const T*>(p) + at);
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = to_f32(v.v[i]);
    }
}

// What is computed from v from here on is computed anew: without this the
// compiler keeps the fp32 forms of a row in 16 bits, twice its registers, from
// one use to the next.
template <typename T, int E>
__device__ __forceinline__ void forget(Pack<T, E>& v) {
    if constexpr (sizeof(v) % 4 == 0) {
        uint32_t w[sizeof(v) / 4];
        __builtin_memcpy(w, &v, sizeof(v));
#pragma unroll
        for (unsigned k = 0; k < sizeof(v) / 4; ++k) asm("" : "+v"(w[k]));
        __builtin_memcpy(&v, w, sizeof(v));
    }
}

template <int kCtrl>
__device__ __forceinline__ float dpp_move(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), kCtrl, 0xf, 0xf, true));
}

// x combined over the team of G lanes (a power of two, at most a wavefront) that
// the lane is in; every lane gets the same bits, since each step combines two
// partial results in either order.
template <int G, typename Op>
__device__ __forceinline__ float team_combine(float x, Op op) {
    if constexpr (G == 16 || G == 32 || G == 64) {
        x = op(x, dpp_move<0x128>(x));  // row_ror:8
        x = op(x, dpp_move<0x124>(x));  // row_ror:4
        x = op(x, dpp_move<0x122>(x));
        x = op(x, dpp_move<0x121>(x));
        if constexpr (G >= 32) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
        if constexpr (G == 64) {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
    } else {
        if constexpr (G == 8) x = op(x, dpp_move<0x141>(x));     // row_half_mirror
        if constexpr (G >= 4) x = op(x, dpp_move<0x4e>(x));      // quad_perm 2,3,0,1
        if constexpr (G >= 2) x = op(x, dpp_move<0xb1>(x));      // quad_perm 1,0,3,2
    }
    return x;
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    return max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kCtrl, 0xf, 0xf, true)));
}

// The largest x of the wavefront's lanes, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = dpp_max<0x121>(dpp_max<0x122>(dpp_max<0x124>(dpp_max<0x128>(x))));
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(r[0], r[1]);
    const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(s[0], s[1]);
}

struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// Lanes of a workgroup whose teams have G: 256, or one team of several wavefronts.
constexpr int team_threads(int G) { return G <= 64 ? 256 : G; }

// N values combined over a team of G lanes.  A team of more than a wavefront is
// the whole workgroup: its wavefronts meet in LDS, in one of two buffers in
// turn, so that one barrier per call is enough (a buffer is written again only
// after the barrier of the call between).
template <int G, int N, typename Op>
struct Team {
    static constexpr int kWaves = G > 64 ? G / 64 : 1;
    float* buffer;  // [2][N][kWaves] of LDS, G > 64 only
    int turn = 0;

    __device__ __forceinline__ explicit Team(float* lds) : buffer(lds) {}

    __device__ __forceinline__ void operator()(float (&x)[N], Op op = Op()) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = team_combine<G < 64 ? G : 64>(x[i], op);
        if constexpr (G > 64) {
            float* slot = buffer + turn * N * kWaves;
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            if (lane == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) slot[i * kWaves + wave] = x[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = team_combine<kWaves>(slot[i * kWaves + (lane & (kWaves - 1))], op);
            turn ^= 1;
        }
    }
};

// A row's columns as a team of G lanes takes them: V vectors of E per lane, the
// v-th of lane l at (v * G + l) * E.  Only the last vector can pass the row's
// end: it then starts at n - E instead (n >= E) and its first `skip` values, which
// another vector has too, count for nothing in sums.
template <int E, int G, int V>
struct Columns {
    int at[V];
    int skip;     // of the last vector; E: none of it counts
    bool last;    // the last vector lies in the row
    __device__ __forceinline__ Columns(int lane, int n) {
#pragma unroll
        for (int v = 0; v < V; ++v) at[v] = (v * G + lane) * E;
        const int c = at[V - 1];
        last = c < n;
        at[V - 1] = c < n - E ? c : n - E;
        skip = last ? c - at[V - 1] : E;
    }
    __device__ __forceinline__ bool counts(int v, int i) const { return v < V - 1 || i >= skip; }
    __device__ __forceinline__ bool inside(int v) const { return v < V - 1 || last; }
};

}  // namespace tca
