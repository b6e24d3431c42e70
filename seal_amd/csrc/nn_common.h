// Pieces shared by the kernels of the quantised, sampled decode (w4_kernels.hip, kv8_kernels.hip, sample_kernels.hip): storage types,
// the exact bf16 planes of an fp32 number, launch checks.
#ifndef NN_COMMON_H
#define NN_COMMON_H
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <exception>
#include <stdint.h>
#include <type_traits>

#include "../../include/sealnn.h"
#include "fmi_internal.h"

#define NNCHK() do { hipError_t e_ = hipGetLastError(); if (e_ != hipSuccess) { fmi_set_error("sealnn launch failed: %s", hipGetErrorString(e_)); return FMI_ERR_HIP; } } while (0)

typedef __hip_bfloat16 bf16;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
// loads of four elements from an address that is only aligned to one (rows of an odd length): gfx950 takes them in one instruction
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

static __device__ __forceinline__ float as_f32(uint32_t u) { return __uint_as_float(u); }
static __device__ __forceinline__ uint32_t as_u32(float f) { return __float_as_uint(f); }

template <typename T> static __device__ __forceinline__ float load1(const T *p);
template <> __device__ __forceinline__ float load1<float>(const float *p) { return *p; }
template <> __device__ __forceinline__ float load1<bf16>(const bf16 *p) { return as_f32((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16); }
template <typename T> static __device__ __forceinline__ void store1(T *p, float v);
template <> __device__ __forceinline__ void store1<float>(float *p, float v) { *p = v; }
template <> __device__ __forceinline__ void store1<bf16>(bf16 *p, float v) { *p = __float2bfloat16(v); }      // (to nearest, ties to even)

// the upper halves of two words as one word: two fp32 numbers truncated to bf16
static __device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// Eight fp32 numbers as three bf16 planes whose sum they ARE: bf16 has fp32's range and 8 of its 24 significant bits, so
//     hi = x truncated,   mid = (x - hi) truncated,   lo = x - hi - mid
// are exact (each difference has 8 significant bits less), and a product against bf16 numbers is three bf16 matrix instructions that
// accumulate what one on fp32 operands would.  (An infinity leaves inf - inf in the lower planes: NaN.)
struct Planes { bf16x8 p[3]; };
static __device__ __forceinline__ void split8(const float x[8], Planes &out)
{
    u32x4 w[3];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = x[2 * i], b = x[2 * i + 1];
        const float ra = a - as_f32(as_u32(a) & 0xffff0000u), rb = b - as_f32(as_u32(b) & 0xffff0000u);
        const float la = ra - as_f32(as_u32(ra) & 0xffff0000u), lb = rb - as_f32(as_u32(rb) & 0xffff0000u);
        w[0][i] = upper_halves(as_u32(a), as_u32(b));
        w[1][i] = upper_halves(as_u32(ra), as_u32(rb));
        w[2][i] = upper_halves(as_u32(la), as_u32(lb));
    }
#pragma unroll
    for (int i = 0; i < 3; i++) out.p[i] = __builtin_bit_cast(bf16x8, w[i]);
}

#endif
