// Element types and wide loads / stores of the sequence-policy operators (gated_scan.hip, rms_norm.hip, distill.hip).
// Tensors are fp32, bf16 or fp16; every sum, state and statistic is fp32; a value is rounded once, to nearest even, when
// it is stored.
#pragma once
#include "common.h"

#define SERL_F32 0      // type codes of the C ABI
#define SERL_BF16 1
#define SERL_F16 2

typedef uint32_t sq_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t sq_u32x4 __attribute__((ext_vector_type(4)));   // native vectors stay in registers
typedef uint16_t sq_u16;
typedef float sq_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 sq_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 sq_f16x2 __attribute__((ext_vector_type(2)));

struct F32 { typedef uint32_t bits; static constexpr int code = SERL_F32; };
struct BF16 { typedef uint16_t bits; static constexpr int code = SERL_BF16; };
struct F16 { typedef uint16_t bits; static constexpr int code = SERL_F16; };

__device__ __forceinline__ float sq_val(F32, uint32_t b) { return __uint_as_float(b); }
__device__ __forceinline__ float sq_val(BF16, uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ float sq_val(F16, uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
__device__ __forceinline__ uint32_t sq_bits(F32, float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint16_t sq_bits(BF16, float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ uint16_t sq_bits(F16, float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

// two packed 16-bit values of a dword, and back
template <typename T> __device__ __forceinline__ void sq_unpack2(uint32_t w, float& a, float& b) {
  a = sq_val(T(), (uint16_t)(w & 0xffffu));
  b = sq_val(T(), (uint16_t)(w >> 16));
}
template <> __device__ __forceinline__ void sq_unpack2<BF16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ uint32_t sq_pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t sq_pack2<BF16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((sq_f32x2){a, b}, sq_bf16x2));
}
template <> __device__ __forceinline__ uint32_t sq_pack2<F16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((sq_f32x2){a, b}, sq_f16x2));
}

// VEC consecutive elements of type T as they lie in memory (VEC * size = a power of two of bytes, naturally aligned; LOOSE: at any
// element, the same instructions, which the hardware takes at any address; STREAM:
// touched once, in whole cache lines, not to be kept in the caches; VEC = 1: one element)
template <typename T, int VEC> struct Raw {
  static constexpr int BYTES = VEC * (int)sizeof(typename T::bits);
  static constexpr int W = BYTES / 4;
  static_assert(BYTES % 4 == 0, "whole dwords");
  uint32_t w[W];
  template <bool LOOSE = false, bool STREAM = false> __device__ __forceinline__ void load(const typename T::bits* p) {
    if constexpr (LOOSE) {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        sq_u32x4 v = {};
        __builtin_memcpy(&v, (const char*)p + 4 * i, W < 4 ? BYTES : 16);
#pragma unroll
        for (int j = 0; j < 4 && i + j < W; ++j) w[i + j] = v[j];
      }
    } else if constexpr (W % 4 == 0) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const sq_u32x4* q = reinterpret_cast<const sq_u32x4*>(p) + i;
        const sq_u32x4 v = STREAM ? __builtin_nontemporal_load(q) : *q;
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else if constexpr (W == 2) {
      const sq_u32x2 v = *reinterpret_cast<const sq_u32x2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else {
      static_assert(W == 1, "1, 2 or 4n dwords");
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  template <bool LOOSE = false, bool STREAM = false> __device__ __forceinline__ void store(typename T::bits* p) const {
    if constexpr (LOOSE) {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        sq_u32x4 v = {};
#pragma unroll
        for (int j = 0; j < 4 && i + j < W; ++j) v[j] = w[i + j];
        __builtin_memcpy((char*)p + 4 * i, &v, W < 4 ? BYTES : 16);
      }
    } else if constexpr (W % 4 == 0) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const sq_u32x4 v = {w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<sq_u32x4*>(p) + i);
        else reinterpret_cast<sq_u32x4*>(p)[i] = v;
      }
    } else if constexpr (W == 2) {
      *reinterpret_cast<sq_u32x2*>(p) = (sq_u32x2){w[0], w[1]};
    } else {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    if constexpr (sizeof(typename T::bits) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) sq_unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void put(const float (&v)[VEC]) {
    if constexpr (sizeof(typename T::bits) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = sq_pack2<T>(v[2 * i], v[2 * i + 1]);
    }
  }
};
template <typename T> struct Raw<T, 1> {
  typename T::bits w;
  template <bool LOOSE = false, bool STREAM = false> __device__ __forceinline__ void load(const typename T::bits* p) { w = *p; }
  template <bool LOOSE = false, bool STREAM = false> __device__ __forceinline__ void store(typename T::bits* p) const { *p = w; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = sq_val(T(), w); }
  __device__ __forceinline__ void put(const float (&v)[1]) { w = sq_bits(T(), v[0]); }
};

// The next get() of r unpacks anew: without this the compiler keeps the 32-bit values of the first one for the later ones,
// twice the registers of a 16-bit type.
template <typename T, int VEC> __device__ __forceinline__ void sq_again(Raw<T, VEC>& r) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int i = 0; i < Raw<T, VEC>::W; ++i) asm volatile("" : "+v"(r.w[i]));
  }
}

// Raw buffer access: a uniform base, a 32-bit byte offset per lane, and the hardware's check against `bytes` (reads behind them
// give 0, writes are dropped), so partial tiles need neither clamped addresses nor branches around loads.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t sq_buffer(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}
// STREAM: the non-temporal hint.
#define SQ_NOWHERE 0x80000000u      // an offset behind every buffer
template <bool STREAM = false, typename T, int VEC> __device__ __forceinline__ void sq_load(Raw<T, VEC>& r, __amdgpu_buffer_rsrc_t b, uint32_t off) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(typename T::bits) == 2) r.w = __builtin_amdgcn_raw_buffer_load_b16(b, off, 0, STREAM ? 2 : 0);
    else r.w = __builtin_amdgcn_raw_buffer_load_b32(b, off, 0, STREAM ? 2 : 0);
  } else if constexpr (Raw<T, VEC>::W == 2) {
    const sq_u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, STREAM ? 2 : 0);
    r.w[0] = v.x; r.w[1] = v.y;
  } else {
    static_assert(VEC == 1 || Raw<T, VEC>::W == 4, "one access");
    const sq_u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, STREAM ? 2 : 0);
    r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
  }
}
template <bool STREAM = false, typename T, int VEC> __device__ __forceinline__ void sq_store(const Raw<T, VEC>& r, __amdgpu_buffer_rsrc_t b, uint32_t off) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(typename T::bits) == 2) __builtin_amdgcn_raw_buffer_store_b16(r.w, b, off, 0, STREAM ? 2 : 0);
    else __builtin_amdgcn_raw_buffer_store_b32(r.w, b, off, 0, STREAM ? 2 : 0);
  } else if constexpr (Raw<T, VEC>::W == 2) {
    __builtin_amdgcn_raw_buffer_store_b64((sq_u32x2){r.w[0], r.w[1]}, b, off, 0, STREAM ? 2 : 0);
  } else {
    static_assert(VEC == 1 || Raw<T, VEC>::W == 4, "one access");
    __builtin_amdgcn_raw_buffer_store_b128((sq_u32x4){r.w[0], r.w[1], r.w[2], r.w[3]}, b, off, 0, STREAM ? 2 : 0);
  }
}

static inline bool sq_aligned(const void* p, int bytes) { return ((uintptr_t)p % (uintptr_t)bytes) == 0; }
#define SQ_STREAM (5ll << 26)       // a call that moves more bytes gains from streaming accesses (the last cache level has 2^28)
static inline int sq_size(int code) { return code == SERL_F32 ? 4 : 2; }

// f over the 16, 32 or 64 lanes that a lane is one of, the same bits in all of them: lane exchanges of the vector ALU (the halves, the
// rows of 16, then rotations within them), a fraction of the latency of shuffles through LDS
// (distillation of 100000 x 64 bf16 97 -> 87 us, 2048 x 131072 224 -> 217).
template <int N> __device__ __forceinline__ uint32_t sq_rotate(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, false);
}
template <int LANES, typename F> __device__ __forceinline__ uint32_t sq_over_lanes(uint32_t v, F f) {
  if constexpr (LANES == 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = f(p[0], p[1]);
  }
  if constexpr (LANES >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(p[0], p[1]);
  }
  v = f(v, sq_rotate<8>(v));
  v = f(v, sq_rotate<4>(v));
  v = f(v, sq_rotate<2>(v));
  return f(v, sq_rotate<1>(v));
}
template <int LANES = 64> __device__ __forceinline__ float sq_wave_sum(float v) {
  return __uint_as_float(sq_over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ float sq_wave_max(float v) {       // NaN lose
  return __uint_as_float(sq_over_lanes<64>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
