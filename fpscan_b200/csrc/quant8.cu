// quantize8 / dequantize8: a tensor kept in 8 bits for the backward pass, in
// blocks of 64 consecutive values (format in quant8.cuh).
//
// Bound by memory: the value's bytes and one more in each direction.  To 8
// bits, four lanes share a block, 16 values each: the block's quotients are
// worked out by every lane (with eight lanes they cost 113 us instead of 85),
// its magnitude is two shuffles, and no shared memory or second pass is
// needed.  32768 x 4096 bf16: to 8 bits 85 us (4.8 TB/s), back 71 us (5.7 TB/s).
#include <algorithm>

#include "internal.h"
#include "quant8.cuh"

namespace fpscan {

namespace {

constexpr int kBlock8 = 64;

struct Quant8Params {
  const void* x;
  void* out;
  int8_t* codes;
  const int8_t* codes_in;
  float* steps;
  const float* steps_in;
  int64_t n;
};

// A 16-byte vector from p; values at or past `left` are 0.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* p, int64_t left FPSCAN_DEBUG_ONLY(, const T* lo, const T* hi)) {
  constexpr int V = Elem<T>::kVec;
  Vec16<T> v;
  v.raw = make_uint4(0, 0, 0, 0);
  FPSCAN_DEBUG_ONLY(if (left > 0 && !in_bounds(p, (left < V ? left : V) * sizeof(T), lo, hi)) return v.raw;)
  if (left >= V) {
    v.raw = *reinterpret_cast<const uint4*>(p);
  } else {
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (c < left) v.e[c] = p[c];
  }
  return v.raw;
}

template <typename T>
__global__ void __launch_bounds__(256) quantize8_kernel(const Quant8Params p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t units = (p.n + kBlock8 - 1) / kBlock8 * 4;  // whole blocks: all lanes of a group stay
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  const T* src = static_cast<const T*>(p.x);
  // the loop's bound is a multiple of 4 lanes, not of 32: the shuffles name their group
  const unsigned mask = 0xfu << (threadIdx.x & 28);
  for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < units; u += step) {
    const int64_t i = u * 16, left = p.n - i;
    constexpr int V = Elem<T>::kVec;
    uint4 raw[16 / V];
#pragma unroll
    for (int j = 0; j < 16 / V; ++j) raw[j] = load_vec(src + i + j * V, left - j * V FPSCAN_DEBUG_ONLY(, src, src + p.n));
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 16 / V; ++j) most = quant8_max<T>(most, quant8_max<T>(raw[j]));
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) most = quant8_max<T>(most, __shfl_xor_sync(mask, most, d));
    const Quant8 q = quant8_block<T>(quant8_bits<T>(most));
    uint32_t w[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      Vec16<T> v;
      v.raw = raw[4 * c / V];
      const T* y = v.e + 4 * c % V;
      w[c] = quant8_codes<T>(q, Elem<T>::load(y[0]), Elem<T>::load(y[1]), Elem<T>::load(y[2]),
                             Elem<T>::load(y[3]));
    }
    // (a block's lanes behind the tensor's end hold nothing)
    FPSCAN_DEBUG_ONLY(if (left > 0 && !in_bounds(p.codes + i, left < 16 ? left : 16, p.codes, p.codes + p.n)) continue;)
    if (left >= 16)
      *reinterpret_cast<uint4*>(p.codes + i) = make_uint4(w[0], w[1], w[2], w[3]);
    else
#pragma unroll
      for (int c = 0; c < 16; ++c)
        if (c < left) p.codes[i + c] = (int8_t)(w[c / 4] >> (8 * (c & 3)));
    if ((u & 3) == 0 FPSCAN_DEBUG_ONLY(
                         && in_bounds<4>(p.steps + u / 4, 4, p.steps, p.steps + (p.n + kBlock8 - 1) / kBlock8)))
      p.steps[u / 4] = q.step;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize8_kernel(const Quant8Params p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t units = (p.n + 7) / 8, step = (int64_t)gridDim.x * blockDim.x;
  T* dst = static_cast<T*>(p.out);
  for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < units; u += step) {
    const int64_t i = u * 8, left = p.n - i;
    FPSCAN_DEBUG_ONLY(
        const int64_t some = left < 8 ? left : 8;
        if (!in_bounds<4>(p.steps_in + u / 8, 4, p.steps_in, p.steps_in + (p.n + kBlock8 - 1) / kBlock8) ||
            !in_bounds<8>(p.codes_in + i, some, p.codes_in, p.codes_in + p.n) ||
            !in_bounds(dst + i, some * sizeof(T), dst, dst + p.n)) continue;)
    const float s = p.steps_in[u / 8];
    if (left >= 8) {
      const uint2 w = *reinterpret_cast<const uint2*>(p.codes_in + i);
      float x[8];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = quant8_value(w.x, c, s);
        x[4 + c] = quant8_value(w.y, c, s);
      }
#pragma unroll
      for (int j = 0; j < 8 / Elem<T>::kVec; ++j)
        *reinterpret_cast<uint4*>(dst + i + j * Elem<T>::kVec) = pack_vec<T>(x + j * Elem<T>::kVec);
    } else {
      for (int c = 0; c < left; ++c) dst[i + c] = Elem<T>::store((float)p.codes_in[i + c] * s);
    }
  }
}

template <typename T>
cudaError_t run8(const Quant8Args& a) {
  Quant8Params p{a.x, a.out, a.codes, a.codes, a.steps, a.steps, a.n};
  const int64_t ctas = (a.n + 2047) / 2048;
  const unsigned grid = (unsigned)std::min<int64_t>(ctas, (int64_t)a.num_sms * 32);
  return a.x != nullptr ? launch_pdl(quantize8_kernel<T>, grid, 256, 0, a.stream, p)
                        : launch_pdl(dequantize8_kernel<T>, grid, 256, 0, a.stream, p);
}

}  // namespace

cudaError_t launch_quant8(const Quant8Args& a) {
  switch (a.dtype) {
    case kF32:
      return run8<float>(a);
    case kF16:
      return run8<__half>(a);
    default:
      return run8<__nv_bfloat16>(a);
  }
}

}  // namespace fpscan
