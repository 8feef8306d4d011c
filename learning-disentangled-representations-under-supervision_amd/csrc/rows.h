// Rows of float or bf16 values in 16-byte pieces, for the kernels that hold a row in registers (layernorm.hip,
// token_loss.hip) and for gradnorm.hip. A row may start at any element boundary (odd widths): the pieces are loaded and
// stored through types of element alignment, which gfx950 executes as one 16-byte access each; the C % E last elements
// go one by one, so no access leaves the row.
#pragma once
#include "common.h"

// load_stream / store_stream mark data that will not be read again before the 256 MB cache has seen its size in other
// data: it then neither pushes out what is wanted nor leaves dirty lines for later reads to wait on. A copy of 512 MB with
// both marks runs at 6.3 TB/s, without them at 5.6 (5.1 to 5.2 with few, long-running workgroups).

namespace cgn_rows {

constexpr int64_t STREAM_BYTES = 128 << 20;  // data from this size on is streamed: half of the cache

struct Bf16 {
    unsigned short bits;
};

typedef unsigned u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4_e4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ float bf16_to_f32(unsigned short h) {
    return __builtin_bit_cast(float, (unsigned)h << 16);
}
// round to nearest, ties to even; a NaN stays a (quiet) NaN
__device__ __forceinline__ unsigned short f32_to_bf16(float f) {
    return __builtin_bit_cast(unsigned short, (__bf16)f);
}

template <typename T>
struct Piece;

template <>
struct Piece<float> {
    static constexpr int E = 4;
    f32x4 v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const f32x4_e4*>(p); }
    __device__ __forceinline__ void load_stream(const float* p) {
        v = __builtin_nontemporal_load(reinterpret_cast<const f32x4_e4*>(p));
    }
    __device__ __forceinline__ void fill(float x) { v = f32x4{x, x, x, x}; }
    __device__ __forceinline__ float get(int e) const { return v[e]; }
    static __device__ __forceinline__ void store(float* p, const float (&o)[E]) {
        *reinterpret_cast<f32x4_e4*>(p) = f32x4{o[0], o[1], o[2], o[3]};
    }
    static __device__ __forceinline__ void store_stream(float* p, const float (&o)[E]) {
        const f32x4_e4 w = {o[0], o[1], o[2], o[3]};
        __builtin_nontemporal_store(w, reinterpret_cast<f32x4_e4*>(p));
    }
    static __device__ __forceinline__ void put(float* p, float x) { *p = x; }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
};

template <>
struct Piece<Bf16> {
    static constexpr int E = 8;
    unsigned v __attribute__((ext_vector_type(4)));
    __device__ __forceinline__ void load(const Bf16* p) { v = *reinterpret_cast<const u32x4_e2*>(p); }
    __device__ __forceinline__ void load_stream(const Bf16* p) {
        v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_e2*>(p));
    }
    __device__ __forceinline__ void fill(float x) {
        const unsigned h = f32_to_bf16(x), w = h | h << 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = w;
    }
    __device__ __forceinline__ float get(int e) const {
        const unsigned w = v[e >> 1];
        return __builtin_bit_cast(float, e & 1 ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ u32x4_e2 pack(const float (&o)[E]) {
        u32x4_e2 w;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{o[2 * e], o[2 * e + 1]}, bf16x2));
        return w;
    }
    static __device__ __forceinline__ void store(Bf16* p, const float (&o)[E]) { *reinterpret_cast<u32x4_e2*>(p) = pack(o); }
    static __device__ __forceinline__ void store_stream(Bf16* p, const float (&o)[E]) {
        __builtin_nontemporal_store(pack(o), reinterpret_cast<u32x4_e2*>(p));
    }
    static __device__ __forceinline__ void put(Bf16* p, float x) { p->bits = f32_to_bf16(x); }
    static __device__ __forceinline__ float one(const Bf16* p) { return bf16_to_f32(p->bits); }
};

// bf16 rows stay packed (two elements a register) from pass to pass over them and are unpacked, and take their
// exponentials, anew: kept, the floats would need twice the registers and halve the waves per CU. The compiler must not
// see that the passes form the same values. (fp32 rows are as they are.)
template <typename T, int NV>
__device__ __forceinline__ void keep_packed(Piece<T> (&q)[NV]) {
    if constexpr (Piece<T>::E == 8) {
#pragma unroll
        for (int j = 0; j < NV; ++j) asm volatile("" : "+v"(q[j].v));
    }
}

// Sum over the G lanes of a group (G a power of two up to the wave); every lane gets it.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

}  // namespace cgn_rows
