// In place of the HIP runtime's header where a kernel's source is compiled for the CPU: the words of the language, and
// the lanes' and the workgroup's operations on a model in which every thread runs by itself and the waves of a workgroup go
// on in random order between barriers (model.cpp). What it shows: reads of LDS that a barrier is missing for, barriers
// that not all threads reach, and, with memory that ends where the data does, reads and writes out of range.
#pragma once
#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <functional>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static

namespace model {
void launch(unsigned grid, unsigned block, const std::function<void()>& kernel);
int thread();                                   // of the workgroup
void barrier();
uint64_t from_lane(uint64_t x, int lane);       // what that lane of the wave has given
uint64_t lanes_with(bool x);
inline int lane() { return thread() & 63; }
template <typename T>
T exchange(T x, int lane) {
  uint64_t u = 0;
  memcpy(&u, &x, sizeof(T));
  u = from_lane(u, lane);
  memcpy(&x, &u, sizeof(T));
  return x;
}
struct ThreadX {
  operator unsigned() const { return (unsigned)thread(); }
};
struct Pair {
  uint32_t v[2];
  uint32_t operator[](int i) const { return v[i]; }
};
inline Pair swapped(uint32_t x, int j) { return {exchange(x, lane() & ~j), exchange(x, lane() | j)}; }
inline int dpp_source(int control, int l) {
  switch (control) {
    case 0x111: case 0x112: case 0x114: case 0x118:                     // row_shr
      return (l & 15) >= control - 0x110 ? l - (control - 0x110) : -1;
    case 0x142: return l >= 16 ? (l & ~15) - 1 : -1;                    // row_bcast:15, to the next row
    case 0x143: return l >= 32 ? 31 : -1;                               // row_bcast:31
    case 0xB1: return l ^ 1;                                            // quad_perm:[1,0,3,2]
    case 0x4E: return l ^ 2;                                            // quad_perm:[2,3,0,1]
    case 0x1B: return l ^ 3;                                            // quad_perm:[3,2,1,0]
    case 0x141: return l ^ 7;                                           // row_half_mirror
    case 0x128: return (l & ~15) | ((l + 8) & 15);                      // row_ror:8
  }
  abort();
}
}  // namespace model

struct Dim {
  unsigned x;
};
extern Dim blockIdx, blockDim;
static const struct {
  model::ThreadX x;
} threadIdx = {};

typedef int hipError_t;
typedef void* hipStream_t;
inline hipError_t hipGetLastError() { return 0; }
struct uint2 {
  uint32_t x, y;
};
struct uint4 {
  uint32_t x, y, z, w;
};
inline uint2 make_uint2(uint32_t x, uint32_t y) { return {x, y}; }
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }
using std::max;
using std::min;

inline void __syncthreads() { model::barrier(); }
template <typename T>
T __shfl_xor(T x, int mask) { return model::exchange(x, model::lane() ^ mask); }
inline unsigned long long __ballot(bool x) { return model::lanes_with(x); }
inline bool __any(bool x) { return model::lanes_with(x) != 0; }
inline int __popcll(unsigned long long x) { return __builtin_popcountll(x); }
inline uint32_t __umulhi(uint32_t x, uint32_t y) { return (uint32_t)((uint64_t)x * y >> 32); }
inline int __clz(int x) { return x ? __builtin_clz((unsigned)x) : 32; }
template <typename T, typename U>
T atomicAdd(T* p, U x) {
  const T old = *p;
  *p = old + (T)x;
  return old;
}
inline uint32_t __float_as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }
inline float __uint_as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
inline long long __double_as_longlong(double x) { return __builtin_bit_cast(long long, x); }
inline double __longlong_as_double(long long x) { return __builtin_bit_cast(double, x); }

// Lanes whose row is masked, or whose source is outside, keep `old`.
inline int __builtin_amdgcn_update_dpp(int old, int x, int control, int rows, int, bool) {
  const int l = model::lane(), source = model::dpp_source(control, l);
  const int y = model::exchange(x, source < 0 ? l : source);
  return source < 0 || !(rows >> (l >> 4) & 1) ? old : y;
}
inline int __builtin_amdgcn_readlane(int x, int lane) { return model::exchange(x, lane); }
#define __builtin_amdgcn_readfirstlane(x) model::exchange(x, 0)
#define __builtin_amdgcn_permlane16_swap(x, y, ...) model::swapped(x, 16)
#define __builtin_amdgcn_permlane32_swap(x, y, ...) model::swapped(x, 32)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __expf(x) expf(x)
#define __builtin_isunordered(a, b) ((a) != (a) || (b) != (b))
// (named in headers, by kernels that are not compiled here)
inline uint32_t __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(uint32_t, float, int) { abort(); }
inline uint32_t __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(uint32_t, float, float, float, int) { abort(); }
