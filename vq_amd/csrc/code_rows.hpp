// Rows of scores as they lie in the registers of a wave or a workgroup.
#pragma once
#include <type_traits>

#include "logprobs.hpp"

namespace vq {

// The codes [lo, hi) of a row in LANES lanes: vector u of a lane holds the VEC codes from lo + (u * LANES + lane) * VEC on, as they are
// stored; what lies behind the end is -inf.
template <typename T, int LANES, int NV> struct Held {
    typedef typename T::Raw Raw;
    static constexpr int VEC = 16 / (int)sizeof(Raw), E = NV * VEC;
    static constexpr uint32_t NONE = sizeof(Raw) == 4 ? 0xff800000u : std::is_same<T, F16>::value ? 0xfc00fc00u : 0xff80ff80u;
    struct __attribute__((packed, aligned(sizeof(Raw)))) Piece {
        uint32_t w[4];
    };
    Piece raw[NV];

    // ONCE: nobody is expected to read the row after this; it passes the caches
    template <bool ONCE = false> static __device__ __forceinline__ Piece fetch(const Raw *s) {
        if constexpr (ONCE)
            return __builtin_bit_cast(Piece, __builtin_nontemporal_load(reinterpret_cast<const AnyWords *>(s)));
        else
            return *reinterpret_cast<const Piece *>(s);
    }
    template <bool ONCE = false> __device__ __forceinline__ void load(const Raw *s, int lo, int hi, int lane) {
        if (lo + LANES * E <= hi) {  // uniform: whole vectors all of them
#pragma unroll
            for (int u = 0; u < NV; ++u) raw[u] = fetch<ONCE>(s + lo + (u * LANES + lane) * VEC);
            return;
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int at = lo + (u * LANES + lane) * VEC;
#pragma unroll
            for (int q = 0; q < 4; ++q) raw[u].w[q] = NONE;
            if (at + VEC <= hi) raw[u] = fetch<ONCE>(s + at);
        }
        // the vector that the row's end cuts
        const int tail = (hi - lo) / VEC, rest = (hi - lo) % VEC;
        if (rest && lane == tail % LANES) {
#pragma unroll
            for (int u = 0; u < NV; ++u)
                if (u == tail / LANES) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v)
                        if (v < rest) put(u, v, s[lo + tail * VEC + v]);
                }
        }
    }
    __device__ __forceinline__ void put(int u, int v, Raw value) {
        if constexpr (sizeof(Raw) == 4)
            raw[u].w[v] = __builtin_bit_cast(uint32_t, value);
        else
            raw[u].w[v >> 1] = v & 1 ? (raw[u].w[v >> 1] & 0xffffu) | (uint32_t)value << 16 : (raw[u].w[v >> 1] & 0xffff0000u) | value;
    }
    __device__ __forceinline__ void drop(int u, int v) {  // a code that counts for nothing from here on
        if constexpr (sizeof(Raw) == 4)
            raw[u].w[v] = NONE;
        else
            raw[u].w[v >> 1] = v & 1 ? (raw[u].w[v >> 1] & 0xffffu) | (NONE & 0xffff0000u) : (raw[u].w[v >> 1] & 0xffff0000u) | (NONE & 0xffffu);
    }
    __device__ __forceinline__ float at(int u, int v) const {
        if constexpr (sizeof(Raw) == 4)
            return __uint_as_float(raw[u].w[v]);
        else
            return T::up((Raw)(v & 1 ? raw[u].w[v >> 1] >> 16 : raw[u].w[v >> 1] & 0xffffu));
    }
};

}  // namespace vq
