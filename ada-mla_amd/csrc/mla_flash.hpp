// Building blocks of the many-row attention kernels (drafted trees, prompts):
// 32x32 MFMA tiles on which every lane owns one query row.
//
// Both products run transposed: S^T = K Q^T and O^T = V^T P^T. The D tile of
// S^T then holds, in lane l, 16 keys of query row l mod 32 (lane l ^ 32 the
// other 16), so the softmax is per lane with one exchange between two lanes;
// and those 16 registers, rounded, are the B operand of O^T as they stand: the
// order of the keys within a product is free, so V^T's rows are read in the
// order that P's registers have. P never leaves the registers and the running
// maximum's factor is one value a lane.
#pragma once

#include <type_traits>
#include <utility>

#include "mla_device.hpp"
#include "mla_internal.hpp"
#include "mla_ring.hpp"

namespace mla {

typedef float floatx16 __attribute__((ext_vector_type(16)));

// D[32x32] += A[32x16] * B[16x32], fp32 accumulate. Lane l supplies
// A[l % 32][8 * (l / 32) + j] and B[8 * (l / 32) + j][l % 32] (j = 0..7) and
// holds D[8 * (i / 4) + 4 * (l / 32) + i % 4][l % 32] (i = 0..15).
__device__ __forceinline__ floatx16 mfma32x32x16(half8 a, half8 b, floatx16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ floatx16 mfma32x32x16(bf16x8 a, bf16x8 b, floatx16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The same product accumulated in ordinary registers, for kernels that fill the
// accumulation registers with something else: other accumulators, or with _acc
// the B operand itself. (The compiler puts all of a kernel's products into
// accumulation registers, and moves what does not fit back and forth.)
// A chain: first (C = 0), next .., then settle, or 12 instructions more and
// in_registers, before anything reads the tile: a product's result may be read 12 issue
// slots after an 8-pass product, which the compiler knows of its own
// products only; nor does it know that an operand which a vector instruction
// wrote may be read 2 slots later. Operands therefore come from LDS or are never
// moved, which a test of the assembly checks. Within a chain each product's
// accumulator is exactly the last one's result, which needs no wait.
#define MLA_MFMA_CHAIN(suffix, type, b_class, instruction)                                  \
    __device__ __forceinline__ void mfma32x32x16_first##suffix(floatx16 &d, type a, type b) \
    {                                                                                       \
        asm volatile(instruction " %0, %1, %2, 0" : "=&v"(d) : "v"(a), b_class(b));         \
    }                                                                                       \
    __device__ __forceinline__ void mfma32x32x16_next##suffix(floatx16 &d, type a, type b)  \
    {                                                                                       \
        asm volatile(instruction " %0, %1, %2, %0" : "+v"(d) : "v"(a), b_class(b));         \
    }
MLA_MFMA_CHAIN(, half8, "v", "v_mfma_f32_32x32x16_f16")
MLA_MFMA_CHAIN(, bf16x8, "v", "v_mfma_f32_32x32x16_bf16")
MLA_MFMA_CHAIN(_acc, half8, "a", "v_mfma_f32_32x32x16_f16")
MLA_MFMA_CHAIN(_acc, bf16x8, "a", "v_mfma_f32_32x32x16_bf16")
#undef MLA_MFMA_CHAIN

__device__ __forceinline__ void mfma_settle(floatx16 &d)
{
    asm volatile("s_nop 15" : "+v"(d));
}

// Keeps an accumulator tile in the accumulation registers across this point,
// so that 16 of them and 144 registers of Q* fit one wave's 512: left to
// itself the compiler moves them into the 256 others for a rescale and spills.
__device__ __forceinline__ void in_accumulators(floatx16 &v)
{
    asm volatile("" : "+a"(v));
}

// A use of v, whatever it holds: what loads it is waited for here.
template <typename V>
__device__ __forceinline__ void in_registers(V &v)
{
    asm volatile("" : "+v"(v));
}

// The same for an operand that stays in accumulation registers.
template <typename V>
__device__ __forceinline__ void in_acc_registers(V &v)
{
    asm volatile("" : "+a"(v));
}

// f over lanes l and l ^ 32, on the VALU (see reduce_over_lane_groups).
template <typename F>
__device__ __forceinline__ float reduce_halves(float v, F f)
{
    const unsigned u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return f(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// The key (within its 32-key block) in register i of a lane of half hl: that
// register's row of the D tile.
__device__ __forceinline__ int key_of_reg(int i, int hl)
{
    return 8 * (i >> 2) + 4 * hl + (i & 3);
}

// Keys in LDS, rows of at least 256 bytes: 16-byte chunk c of row r sits at c
// ^ key_swizzle(r). Both reads are then free of bank conflicts: a product's row
// reads take 16 lanes, one chunk of 16 rows in a row, at a time, and all 16 places
// differ; a transpose read takes 32 lanes, 4 chunks of 4 rows in a row, and those 4
// rows differ in the upper two bits of their place.
__device__ __forceinline__ int key_swizzle(int r)
{
    return 4 * (r & 3) + ((r >> 2) & 3);
}

// P's registers 8 a .. 8 a + 7, rounded to the type of V: the B operand of keys 16 a ..
// 16 a + 15 of its block. P is in [0, 2^8] and the rounding at most half a
// step of each term; the sums of P that normalise the result stay in fp32. (The
// rest of P as a second operand would double the second product.)
template <typename E>
__device__ __forceinline__ typename Vec<E>::v8 p_operand(const float *p)
{
    typename Vec<E>::v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = (E)p[i];
    return v;
}

// Whether a 16-bit value is an infinity or a NaN.
template <typename E>
__device__ __forceinline__ bool not_finite(unsigned short bits)
{
    const unsigned e = __is_same(E, _Float16) ? 0x7c00u : 0x7f80u;
    return (bits & e) == e;
}

typedef unsigned short ushort2x __attribute__((ext_vector_type(2)));

// The larger of both 16-bit halves, each by itself.
__device__ __forceinline__ unsigned max_u16x2(unsigned a, unsigned b)
{
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(ushort2x, a),
                                                                  __builtin_bit_cast(ushort2x, b)));
}

// 16 bytes per lane from base + off + kAdd + kOffset into LDS at lds + kLds +
// kOffset + 16 * lane (the instruction's own offset counts for both), in three
// instructions: a wave that has a SIMD to itself issues one every 5 to 9
// cycles, some four beside each 32-cycle product. m0, which carries the LDS address, is
// left changed: nothing else in a kernel that calls this uses it, which a test of the
// assembly checks. The addition stands between the write of m0 and its use, which
// needs one slot there.
template <int kAdd, int kLds, int kOffset>
__device__ __forceinline__ void stream_to_lds16(const void *base, int off, unsigned lds)
{
    int at;
    asm volatile("s_add_u32 m0, %3, %4\n\t"
                 "v_add_u32 %0, %5, %1\n\t"
                 "global_load_lds_dwordx4 %0, %2 offset:%6"
                 : "=&v"(at) : "v"(off), "s"(base), "s"(lds), "n"(kLds), "n"(kAdd), "n"(kOffset) : "memory", "scc");
}

// f(0), f(1), .., each with its index as a constant.
template <typename F, int... kIs>
__device__ __forceinline__ void for_constants(F f, std::integer_sequence<int, kIs...>)
{
    (f(std::integral_constant<int, kIs>{}), ...);
}

__device__ __forceinline__ unsigned lds_address(const void *p)
{
    return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)p);
}

// An address that is the same in all lanes, into scalar registers.
template <typename T>
__device__ __forceinline__ const T *wave_uniform(const T *p)
{
    const uint64_t u = (uint64_t)(uintptr_t)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
    return (const T *)(uintptr_t)((uint64_t)hi << 32 | lo);
}

// A load of what the kernel does not write, at a wave-uniform address, by the
// scalar unit: a vector load would be waited for with vmcnt, behind every
// global->LDS load in flight.
template <typename T>
__device__ __forceinline__ T scalar_load(const T *p)
{
    return *(const __attribute__((address_space(4))) T *)p;
}

// A read, a write, and a transpose read (lds_read_tr16), at an LDS byte address.
template <typename T>
__device__ __forceinline__ T lds_load(unsigned addr)
{
    return *(const MLA_LDS T *)(uintptr_t)addr;
}

template <typename T>
__device__ __forceinline__ void lds_store(unsigned addr, T v)
{
    *(MLA_LDS T *)(uintptr_t)addr = v;
}

template <typename E>
__device__ __forceinline__ typename Vec<E>::v4 lds_load_tr16(unsigned addr)
{
    return __builtin_bit_cast(typename Vec<E>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MLA_LDS shortx4 *)(uintptr_t)addr));
}

}  // namespace mla
