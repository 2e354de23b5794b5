// Gated delta rule token by token, for one or a few tokens per sequence
// (sm_100a): the form that serving calls once per step.
//
//     S <- a S + beta (v - a S k) k^T,   o = scale S q       (a = exp(log_decay))
//
// The work is the state's bytes: 4 dk dv read and written per head, against
// about 7 flops for each of its elements, so this runs on plain fp32
// arithmetic and is bound by memory.  Rows of the state (one per value) are
// independent.  Eight lanes share a row, each with dk / 8 of its elements in
// 16-byte vectors (128 contiguous bytes per group and load); a thread holds
// kRows rows so that all its loads are in flight at once.  The two sums that
// need the old state, k.S and q.S, are reduced together in three shuffles,
// and q.(S + u k) follows from them and q.k without a second pass.  The state is
// read and written with the hint that it is used once: 198 -> 171 us for 256
// sequences of 32 heads, dk = dv = 128 (6.3 TB/s); four rows per thread 192 us.
#include "delta.cuh"
#include "internal.h"

namespace fpscan {

namespace {

struct StepParams {
  const void* q;
  const void* k;
  const void* v;
  const void* log_decay;
  const void* beta;
  const float* initial;
  float* final_state;
  void* out;
  int64_t L;
  int key_heads, heads, dk, dv, blocks;  // blocks: CTAs along dv
  float scale;
  int64_t batch;  // bounds checks of debug builds
};

constexpr int kStepThreads = 128;
constexpr int kStepRows = 2;                                     // rows of the state per thread
constexpr int kStepCta = kStepThreads / 8 * kStepRows;           // rows per CTA

// Four consecutive elements as fp32.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
}
__device__ __forceinline__ float dot4(const float4& a, const float4& b, float s) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s))));
}

// VEC: 16-byte vectors of a row per lane (dk <= 32 VEC).
template <typename T, int VEC>
__global__ void __launch_bounds__(kStepThreads) delta_step_kernel(const StepParams p) {
  const int tid = threadIdx.x, part = tid & 7;
  const int64_t bh = blockIdx.x / p.blocks;
  const int row0 = (int)(blockIdx.x - bh * p.blocks) * kStepCta + (tid >> 3);
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  pdl_wait();
  pdl_launch_dependents();
  FPSCAN_DEBUG_ONLY(const int64_t n_tok = p.batch * p.L, n_state = p.batch * p.heads * p.dv * p.dk;)

  float4 S[kStepRows][VEC];
#pragma unroll
  for (int r = 0; r < kStepRows; ++r) {
    const int row = row0 + r * (kStepThreads / 8);
    const float* src = p.initial + (bh * p.dv + row) * p.dk;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = (i * 8 + part) * 4;
      S[r][i] = p.initial != nullptr && row < p.dv && c < p.dk FPSCAN_DEBUG_ONLY(
                                                                  && in_bounds(src + c, 16, p.initial, p.initial + n_state))
                    ? __ldcs(reinterpret_cast<const float4*>(src + c))
                    : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  for (int64_t t = 0; t < p.L; ++t) {
    const int64_t tok = b * p.L + t;
    const T* kp = static_cast<const T*>(p.k) + (tok * p.key_heads + hk) * p.dk;
    const T* qp = static_cast<const T*>(p.q) + (tok * p.key_heads + hk) * p.dk;
    float4 k[VEC], q[VEC];
    float qk = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = (i * 8 + part) * 4;
      k[i] = q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < p.dk FPSCAN_DEBUG_ONLY(
                       && within<T, 4 * sizeof(T)>(kp + c, 4, p.k, n_tok * p.key_heads * p.dk)
                       && within<T, 4 * sizeof(T)>(qp + c, 4, p.q, n_tok * p.key_heads * p.dk))) {
        k[i] = load4(kp + c);
        q[i] = load4(qp + c);
      }
      qk = dot4(k[i], q[i], qk);
    }
    FPSCAN_DEBUG_ONLY(
        if (!within<T, sizeof(T)>(static_cast<const T*>(p.log_decay) + tok * p.heads + h, 1, p.log_decay, n_tok * p.heads) ||
            !within<T, sizeof(T)>(static_cast<const T*>(p.beta) + tok * p.heads + h, 1, p.beta, n_tok * p.heads)) return;)
    const float a = expf(Elem<T>::load(static_cast<const T*>(p.log_decay)[tok * p.heads + h]));
    const float beta = Elem<T>::load(static_cast<const T*>(p.beta)[tok * p.heads + h]);
    float v[kStepRows], sk[kStepRows], sq[kStepRows];
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      const int row = row0 + r * (kStepThreads / 8);
      v[r] = row < p.dv FPSCAN_DEBUG_ONLY(
                 && within<T, sizeof(T)>(static_cast<const T*>(p.v) + (tok * p.heads + h) * p.dv + row, 1, p.v,
                                         n_tok * p.heads * p.dv))
                 ? Elem<T>::load(static_cast<const T*>(p.v)[(tok * p.heads + h) * p.dv + row])
                 : 0.f;
      sk[r] = sq[r] = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        S[r][i].x *= a;
        S[r][i].y *= a;
        S[r][i].z *= a;
        S[r][i].w *= a;
        sk[r] = dot4(S[r][i], k[i], sk[r]);
        sq[r] = dot4(S[r][i], q[i], sq[r]);
      }
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
      qk += __shfl_xor_sync(0xffffffffu, qk, d);
#pragma unroll
      for (int r = 0; r < kStepRows; ++r) {
        sk[r] += __shfl_xor_sync(0xffffffffu, sk[r], d);
        sq[r] += __shfl_xor_sync(0xffffffffu, sq[r], d);
      }
    }
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      const int row = row0 + r * (kStepThreads / 8);
      const float u = beta * (v[r] - sk[r]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        S[r][i].x = fmaf(u, k[i].x, S[r][i].x);
        S[r][i].y = fmaf(u, k[i].y, S[r][i].y);
        S[r][i].z = fmaf(u, k[i].z, S[r][i].z);
        S[r][i].w = fmaf(u, k[i].w, S[r][i].w);
      }
      if (part == 0 && row < p.dv FPSCAN_DEBUG_ONLY(
                           && within<T, sizeof(T)>(static_cast<T*>(p.out) + (tok * p.heads + h) * p.dv + row, 1, p.out,
                                                   n_tok * p.heads * p.dv)))
        static_cast<T*>(p.out)[(tok * p.heads + h) * p.dv + row] =
            Elem<T>::store(p.scale * fmaf(u, qk, sq[r]));
    }
  }
  if (p.final_state == nullptr) return;
#pragma unroll
  for (int r = 0; r < kStepRows; ++r) {
    const int row = row0 + r * (kStepThreads / 8);
    float* dst = p.final_state + (bh * p.dv + row) * p.dk;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = (i * 8 + part) * 4;
      if (row < p.dv && c < p.dk FPSCAN_DEBUG_ONLY(
                            && in_bounds(dst + c, 16, p.final_state, p.final_state + n_state)))
        __stcs(reinterpret_cast<float4*>(dst + c), S[r][i]);
    }
  }
}

template <typename T>
cudaError_t step_t(const DeltaArgs& a, const StepParams& p) {
  const unsigned grid = (unsigned)(a.batch * a.heads * p.blocks);
  switch ((a.dk + 31) / 32) {
    case 1:
      return launch_pdl(delta_step_kernel<T, 1>, grid, kStepThreads, 0, a.stream, p);
    case 2:
      return launch_pdl(delta_step_kernel<T, 2>, grid, kStepThreads, 0, a.stream, p);
    case 3:
      return launch_pdl(delta_step_kernel<T, 3>, grid, kStepThreads, 0, a.stream, p);
    default:
      return launch_pdl(delta_step_kernel<T, 4>, grid, kStepThreads, 0, a.stream, p);
  }
}

}  // namespace

cudaError_t launch_delta_step(const DeltaArgs& a) {
  StepParams p{a.q, a.k, a.v, a.log_decay, a.beta, a.initial, a.final_state, a.out, a.seqlen,
               (int)a.key_heads, (int)a.heads, (int)a.dk, (int)a.dv,
               (int)((a.dv + kStepCta - 1) / kStepCta), a.scale, a.batch};
  switch (a.dtype) {
    case kF32:
      return step_t<float>(a, p);
    case kF16:
      return step_t<__half>(a, p);
    default:
      return step_t<__nv_bfloat16>(a, p);
  }
}

}  // namespace fpscan
