// Shared by the token-policy operators (embed.hip, recurrence.hip, log_probs.hip): element types,
// wide accesses at element alignment, and the device guard of their C entries.
#pragma once
#include "common.hpp"

namespace pa {
namespace seq {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Restores the caller's current device: the operators run on the device of their tensors, which
// need not be the current one (a default stream is NULL on every device and names none).
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) : prev_(-1), rc_(PA_OK) {
    int cur = -1;
    hipError_t e = hipGetDevice(&cur);
    if (e == hipSuccess && cur != device) {
      e = hipSetDevice(device);
      if (e == hipSuccess) prev_ = cur;
    }
    if (e != hipSuccess) {
      set_error("device %d: %s", device, hipGetErrorString(e));
      (void)hipGetLastError();      // or the caller's next call would report it
      rc_ = PA_ERR_HIP;
    }
  }
  ~DeviceGuard() {
    if (prev_ >= 0) (void)hipSetDevice(prev_);
  }
  int status() const { return rc_; }

 private:
  int prev_, rc_;
};

#define PA_ON_DEVICE(device)              \
  ::pa::seq::DeviceGuard _guard(device);  \
  if (_guard.status() != PA_OK) return _guard.status()

// N elements of T in registers, as 32-bit words.  Loads and stores assume no more than the element's
// own alignment (gfx950 global accesses may be unaligned), so rows of odd lengths, slices of a wider
// projection and offsets of odd elements take the same wide accesses as aligned ones.
template <typename T, int N>
struct Pack {
  static constexpr int WORDS = N * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
};

template <int BYTES, int N> struct Words;
template <> struct Words<4, 4> { typedef uint32_t U __attribute__((ext_vector_type(4), aligned(4), may_alias)); };
template <> struct Words<2, 4> { typedef uint32_t U __attribute__((ext_vector_type(4), aligned(2), may_alias)); };
template <> struct Words<4, 2> { typedef uint32_t U __attribute__((ext_vector_type(2), aligned(4), may_alias)); };
template <> struct Words<2, 1> { typedef uint32_t U __attribute__((ext_vector_type(1), aligned(2), may_alias)); };
template <> struct Words<2, 2> { typedef uint32_t U __attribute__((ext_vector_type(2), aligned(2), may_alias)); };

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  constexpr int W = Pack<T, N>::WORDS < 4 ? Pack<T, N>::WORDS : 4;      // words per access
  typedef typename Words<(int)sizeof(T), W>::U U;
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < Pack<T, N>::WORDS; i += W) {
    const U u = *reinterpret_cast<const U*>(p + i * 4 / (int)sizeof(T));
#pragma unroll
    for (int k = 0; k < W; ++k) r.w[i + k] = u[k];
  }
  return r;
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& r) {
  constexpr int W = Pack<T, N>::WORDS < 4 ? Pack<T, N>::WORDS : 4;
  typedef typename Words<(int)sizeof(T), W>::U U;
#pragma unroll
  for (int i = 0; i < Pack<T, N>::WORDS; i += W) {
    U u;
#pragma unroll
    for (int k = 0; k < W; ++k) u[k] = r.w[i + k];
    *reinterpret_cast<U*>(p + i * 4 / (int)sizeof(T)) = u;
  }
}

// the first `n` < N elements of a row's last, partial pack; the others are zero / stay unwritten
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_part(const T* p, int n) {
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < Pack<T, N>::WORDS; ++i) r.w[i] = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) {
      if constexpr (sizeof(T) == 4)
        r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
      else
        r.w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
    }
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_part(T* p, const Pack<T, N>& r, int n) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) {
      if constexpr (sizeof(T) == 4)
        reinterpret_cast<uint32_t*>(p)[i] = r.w[i];
      else
        reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(r.w[i / 2] >> (16 * (i & 1)));
    }
}

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& r, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(r.w[i]);
    } else if constexpr (__is_same(T, bf16_t)) {
      f[i] = __uint_as_float((i & 1) ? (r.w[i / 2] & 0xffff0000u) : (r.w[i / 2] << 16));
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, r.w[i / 2]);
      f[i] = (float)((i & 1) ? h.y : h.x);
    }
  }
}

// round to nearest even, the one rounding of a result (overflow to infinity as in a torch cast)
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float (&f)[N]) {
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < Pack<T, N>::WORDS; ++i) {
    if constexpr (sizeof(T) == 4) {
      r.w[i] = __float_as_uint(f[i]);
    } else if constexpr (__is_same(T, bf16_t)) {
      f32x2 p; p.x = f[2 * i]; p.y = f[2 * i + 1];
      r.w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
    } else {
      f16x2 p; p.x = (f16_t)f[2 * i]; p.y = (f16_t)f[2 * i + 1];
      r.w[i] = __builtin_bit_cast(uint32_t, p);
    }
  }
  return r;
}

static inline int elem_size(int dt) {
  return dt == PA_F32 ? 4 : (dt == PA_BF16 || dt == PA_F16) ? 2 : 0;
}

}  // namespace seq
}  // namespace pa
