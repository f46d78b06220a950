// lm_common.hpp -- what the training operators share: errors, types, Philox, row I/O, reductions.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>

#include "../../../include/dion_lm.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------------------------- errors
static thread_local char g_err[512];

static int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
static int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

static int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(DION_E_LAUNCH, "%s: %s", what, hipGetErrorString(e));
  return DION_OK;
}

static inline long ceil_div(long a, long b) { return (a + b - 1) / b; }
static inline long round_up(long a, long b) { return ceil_div(a, b) * b; }
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static inline bool is_float_dtype(int d) { return d == DION_DTYPE_F32 || d == DION_DTYPE_BF16; }

// ------------------------------------------------------------------------------- bf16
struct bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float bf16_to_f32(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
// round to nearest even, NaN stays NaN
__device__ __forceinline__ uint16_t f32_to_bf16(float x) {
  const __bf16 b = static_cast<__bf16>(x);
  uint16_t r;
  __builtin_memcpy(&r, &b, 2);
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return static_cast<uint32_t>(f32_to_bf16(lo)) | (static_cast<uint32_t>(f32_to_bf16(hi)) << 16);
}

// fp16 halves of a word, rounded to nearest even (subnormals kept)
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const _Float16 h[2] = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
  uint32_t r;
  __builtin_memcpy(&r, h, 4);
  return r;
}
__device__ __forceinline__ float f16_lo(uint32_t w) {
  _Float16 h[2];
  __builtin_memcpy(h, &w, 4);
  return static_cast<float>(h[0]);
}
__device__ __forceinline__ float f16_hi(uint32_t w) {
  _Float16 h[2];
  __builtin_memcpy(h, &w, 4);
  return static_cast<float>(h[1]);
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return bf16_to_f32(x.bits); }
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else return T{f32_to_bf16(x)};
}

// N consecutive elements (16 bytes, or 8 floats) at any element's address: gfx950 takes wide accesses at
// any alignment, and the types say so to the compiler.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

template <int N, typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 q = *reinterpret_cast<const f32x4_any*>(p + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i + k] = q[k];
    }
  } else {
    static_assert(N == 8, "bf16 vectors are 16 bytes");
    const u32x4 q = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(q[k] << 16);
      v[2 * k + 1] = __uint_as_float(q[k] & 0xFFFF0000u);
    }
  }
}
template <int N, typename T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4_any*>(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  } else {
    u32x4 q;
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<u32x4_any*>(p) = q;
  }
}
// 8 elements of a row of `cols` from column c on, c < cols; past the end 0, and nothing is stored there.
// !RAGGED: cols is a multiple of 8, and no branch keeps a kernel's loads apart (the norm's backward of
// 8192 x 4096 takes 73 us with the branch and 63 without).
template <bool RAGGED = true, typename T>
__device__ __forceinline__ void load8(const T* row, int c, int cols, float* v) {
  if (!RAGGED || c + 8 <= cols) {
    load_vec<8>(row + c, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? to_f32(row[c + k]) : 0.0f;
  }
}
template <bool RAGGED = true, typename T>
__device__ __forceinline__ void store8(T* row, int c, int cols, const float* v) {
  if (!RAGGED || c + 8 <= cols) {
    store_vec<8>(row + c, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < cols) row[c + k] = from_f32<T>(v[k]);
  }
}

// ------------------------------------------------------------------------------- reductions
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ------------------------------------------------------------------------------- Philox4x32-10
struct DropArgs {
  uint64_t seed, offset;
  const uint64_t* device;
  uint32_t threshold;  // words below it are dropped
  int all;             // p rounds to 1: every element is dropped
  float scale;         // fp32(1 / (1 - p))
};

static DropArgs drop_args(double p, const DionRng* rng) {
  DropArgs a;
  memset(&a, 0, sizeof(a));
  a.scale = 1.0f;
  if (p <= 0.0 || rng == nullptr) return a;
  a.seed = rng->seed;
  a.offset = rng->offset;
  a.device = rng->device;
  const double t = floor(p * 4294967296.0 + 0.5);
  a.all = t >= 4294967296.0;
  a.threshold = a.all ? 0xFFFFFFFFu : static_cast<uint32_t>(t);
  a.scale = a.all ? 0.0f : static_cast<float>(1.0 / (1.0 - p));
  return a;
}

struct Key {
  uint32_t k0, k1, o0, o1;
};
__device__ __forceinline__ Key philox_key(const DropArgs& a) {
  const uint64_t s = a.device ? a.device[0] : a.seed, o = a.device ? a.device[1] : a.offset;
  return Key{static_cast<uint32_t>(s), static_cast<uint32_t>(s >> 32), static_cast<uint32_t>(o),
             static_cast<uint32_t>(o >> 32)};
}
__device__ __forceinline__ void philox4(const Key& key, uint64_t group, uint32_t out[4]) {
  uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32), c2 = key.o0, c3 = key.o1;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c1 = static_cast<uint32_t>(b);
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0;
  out[1] = c1;
  out[2] = c2;
  out[3] = c3;
}
// x * scale where kept, 0 where dropped (a selection: a dropped NaN or infinity is 0 too)
__device__ __forceinline__ float drop1(float x, uint32_t word, const DropArgs& a) {
  return word >= a.threshold && !a.all ? __fmul_rn(x, a.scale) : 0.0f;
}
// N elements that start at element e, a multiple of 4
template <int N>
__device__ __forceinline__ void drop_groups(float* v, uint64_t e, const Key& key, const DropArgs& a) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    philox4(key, (e + i) >> 2, w);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i + k] = drop1(v[i + k], w[k], a);
  }
}
// 8 elements that start at any element (the same e % 4 for the whole wave; !RAGGED: a multiple of 4)
template <bool RAGGED>
__device__ __forceinline__ void drop8(float* v, uint64_t e, const Key& key, const DropArgs& a) {
  const int off = __builtin_amdgcn_readfirstlane(static_cast<int>(e) & 3);
  if (!RAGGED || off == 0) {
    drop_groups<8>(v, e, key, a);
    return;
  }
  uint32_t w[12];
#pragma unroll
  for (int i = 0; i < 3; ++i) philox4(key, (e >> 2) + i, w + 4 * i);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = drop1(v[k], off == 1 ? w[k + 1] : off == 2 ? w[k + 2] : w[k + 3], a);
}
__device__ __forceinline__ void drop_one(float* v, uint64_t e, const Key& key, const DropArgs& a) {
  uint32_t w[4];
  philox4(key, e >> 2, w);
  const uint32_t i = static_cast<uint32_t>(e) & 3u;
  *v = drop1(*v, i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3], a);
}
