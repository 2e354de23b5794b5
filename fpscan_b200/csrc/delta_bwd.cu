// Gated delta rule, backward (sm_100a).  With the chunk's N, P, E, S0 of
// delta.cuh (recomputed by the forward kernels from the inputs) and dS the
// gradient of the state leaving the chunk:
//     F  = P^T dO + beta exp(G_C - G) K dS^T,    dV = N^T F,
//     dS0 = exp(G_C) dS + scale (exp(G) dO)^T Q - (exp(G) dV)^T K      (sequential)
// and then, for every chunk by itself, with H = tril(dO E^T), X = tril(dV E^T, -1),
// Hs = scale D H, Xd = D X:
//     dQ = scale exp(G) dO S0 + Hs diag(beta) K,
//     dK = diag(beta) W + R,  R = -exp(G) dV S0 - Xd diag(beta) K,
//          W = Hs^T Q - Xd^T K + exp(G_C - G) E dS,
//     dbeta_i = k_i . W_i,
//     dlog_decay_t = sum_{i >= t > j} A_ij + sum_{i >= t} reads_i + sum_{j < t} writes_j
//                    + exp(G_C) <S0, dS>,
//          A_ij = beta_j (Hs_ij q_i.k_j - Xd_ij k_i.k_j),
//          reads_i = q_i.(scale exp(G_i) S0^T dO_i) - k_i.(exp(G_i) S0^T dV_i),
//          writes_j = beta_j k_j.(exp(G_C - G_j) dS^T E_j).
// beta and k scale a write alike, hence dbeta: no quotient of a gradient by
// beta or by a decay appears, so zeros of both are harmless.  dlog_decay_t has
// what crosses t and nothing else, and every term carries its own decay: what a
// strong decay or a reset leaves of it is as accurate as any other.  (The sums
// over i >= t of q_i.dQ_i + k_i.R_i - beta_i dbeta_i, plus <S_C, dS>, are the
// same number, but there everything behind t appears twice with opposite
// signs, rounded twice, and drowns it: half of it was noise at a log_decay of
// -10.)
//
//   delta_rev_kernel    from the last chunk to the first, as
//                       delta_scan_kernel; writes dV, and dV, dO, dS as parts.
//   delta_grad_tc_kernel, delta_grad_kernel
//                       the rest, every (chunk, head) by itself: for results
//                       of 16 and of 32 bits.
//   delta_group_kernel  sums dQ, dK over the heads that share a key head, in
//                       a fixed order.
#include <algorithm>

#include "delta.cuh"
#include "internal.h"

namespace fpscan {

template <typename T, int LV>
cudaError_t delta_fwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb,
                           bool keep);

namespace {

// ------------------------------------------------------------------ along the chunks, backwards
struct RevParams {
  const __nv_bfloat16* kq_tiles;
  const void* grad;           // dO
  const __nv_bfloat16* npn;
  const float* vecs;
  const float* grad_final;
  float* dinitial;
  void* dv_out;
  __nv_bfloat16* do_parts;    // strips [head][chunk][dv / 16][NP][64][16]
  __nv_bfloat16* dv_parts;    //        [head][chunk][dv / 16][NS][64][16]
  __nv_bfloat16* ds_parts;    //        [head][chunk][dv / 16][NS][128][16]
  int64_t L, chunks;
  int key_heads, heads, dk, dv, slices;
  float scale;
  int64_t nb;  // sequences (bounds checks of debug builds)
};

constexpr int kRevThreads = 256;

// As delta_scan_kernel, three products per chunk for 2 C values:
//     K dS                                    -> Y,
//     [N; PN]^T [beta exp(G_C - G) Y; dO]     -> dV, since P^T dO enters F and
//                                                N^T P^T = (P N)^T,
//     [K; Q]^T [-exp(G) dV; scale exp(G) dO]  -> the sum that joins dS.
// Both operands of the last two are stacked to 128 rows of k.  The warps of
// tensor memory lanes 0..63 work on Y and dV, those of 64..127 on dO; the
// second product's 64 rows are computed twice over (an operand whose next 64
// rows are the same ones), so that the latter find dV in their lanes too and
// write it out.  4 x 4096 tokens of 16 heads, dk = dv = 128, bf16: 283 us, 1.1
// GB at 4 TB/s (the parts it writes for the gradients are half of it); 2 x
// 2048: 87 us, 32 steps one after another.
template <typename T, int LV, int C>
struct RevCfg {
  static constexpr int NP = kParts<T>;
  static constexpr int NS = LV + 1;
  static constexpr int kKQ = NP * kTileKQ;
  static constexpr int kNPN = NS * 2 * kMatBytes;
  static constexpr int kPart = 128 * 4 * C;    // of dS; of the stacked operands
  static constexpr int kVec = 3 * kChunk * 4;  // enter, leave, beta
  // The stacked operand may lie over dS's parts: they are used up by the
  // first product.  It does where the room is short.
  static constexpr int kRoom = 227 * 1024 - 2 * 1024;
  static constexpr int kFixed = kNPN + 2 * NS * kPart + NextRow<T, C>::kBytes;
  static constexpr bool kOver = kFixed + kKQ + kVec > kRoom;
  static constexpr int kBody = kOver ? kFixed - NS * kPart : kFixed;
  static constexpr int kSt = kBody + 2 * (kKQ + kVec) <= kRoom ? 2 : 1;  // stages of K, Q
  static constexpr int oNPN = kSt * kKQ, oS = oNPN + kNPN, oE = kOver ? oS : oS + NS * kPart;
  static constexpr int oRow = oE + NS * kPart, oVec = oRow + NextRow<T, C>::kBytes;
  static constexpr int kSmem = oVec + kSt * kVec + 1024;
  static_assert(kSmem + 1024 <= 227 * 1024);
};

template <typename T, int LV, int C>
__global__ void __launch_bounds__(kRevThreads, 1) delta_rev_kernel(const RevParams p) {
  using Cfg = RevCfg<T, LV, C>;
  constexpr int kTmem = kTmemColumns<LV, C>;
  constexpr int NP = Cfg::NP, NS = Cfg::NS;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sm0 = smem_addr(dsm);
  const uint32_t s_npn = sm0 + Cfg::oNPN, s_s = sm0 + Cfg::oS, s_e = sm0 + Cfg::oE;
  __shared__ __align__(8) uint64_t full_kq[2], full_n, done[3];
  __shared__ uint32_t s_tmem;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform
  const int quad = warp & 3, col0 = (warp >> 2) * C;  // tensor memory lanes 32 quad.., columns
  const bool is_y = quad < 2;                          // Y and dV; else dO
  const int tok = (quad & 1) * 32 + lane;              // this thread's token
  const int dk = quad * 32 + lane;                     // and row of the state
  const int64_t bh = blockIdx.x / p.slices;
  const int slice = (int)(blockIdx.x - bh * p.slices);
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int dv0 = slice * 2 * C + col0;
  const int nval = min(C, p.dv - dv0);  // values of this thread's C that exist (may be <= 0)
  const int strips = (p.dv + 15) / 16;
  const int64_t vstride = (int64_t)p.heads * p.dv;
  const int64_t tile = (b * p.key_heads + hk) * p.chunks, unit0 = bh * p.chunks;
  FPSCAN_DEBUG_ONLY(const int64_t n_units = p.nb * p.heads * p.chunks, n_tiles = p.nb * p.key_heads * p.chunks,
                    n_v = p.nb * p.L * vstride, n_state = p.nb * p.heads * p.dv * p.dk;)

  if (tid == 0) {
    mbar_init(&full_kq[0], 1);
    mbar_init(&full_kq[1], 1);
    mbar_init(&full_n, 1);
    for (int i = 0; i < 3; ++i) mbar_init(&done[i], 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&s_tmem)), "n"(kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = s_tmem, tmem2 = tmem + NS * 2 * C;  // first and third product; second
  const uint32_t my_tmem = tmem + ((uint32_t)(quad * 32) << 16) + col0;
  pdl_wait();
  pdl_launch_dependents();

  // step d handles chunk chunks - 1 - d
  // Copies are issued by an elected lane of a converged warp (a lone thread of
  // a divergent branch takes over 100 cycles for each).
  const bool loads = warp == kRevThreads / 32 - 1;
  auto load_kq = [&](int64_t d) {
    __syncwarp();
    const int64_t c = p.chunks - 1 - d;
    const int s = (int)(d % Cfg::kSt);
    if (elect_one()) {
      mbar_expect_tx(&full_kq[s], Cfg::kKQ + Cfg::kVec);
      // (a copy left out: the wait for it gives up and is recorded too)
      FPSCAN_DEBUG_ONLY(if (within<char>(p.kq_tiles + (tile + c) * (Cfg::kKQ / 2), Cfg::kKQ, p.kq_tiles, n_tiles * Cfg::kKQ) &&
                            within<float>(p.vecs + (unit0 + c) * (kVecCount * kChunk), Cfg::kVec / 4, p.vecs,
                                          n_units * (kVecCount * kChunk))) {)
      bulk_in(sm0 + s * Cfg::kKQ, p.kq_tiles + (tile + c) * (Cfg::kKQ / 2), Cfg::kKQ, &full_kq[s]);
      bulk_in(sm0 + Cfg::oVec + s * Cfg::kVec, p.vecs + (unit0 + c) * (kVecCount * kChunk), Cfg::kVec,
              &full_kq[s]);
      FPSCAN_DEBUG_ONLY(})
    }
    __syncwarp();
  };
  auto load_n = [&](int64_t d) {
    __syncwarp();
    if (elect_one()) {
      mbar_expect_tx(&full_n, Cfg::kNPN);
      FPSCAN_DEBUG_ONLY(if (within<char>(p.npn + (unit0 + p.chunks - 1 - d) * (Cfg::kNPN / 2), Cfg::kNPN, p.npn,
                                         n_units * Cfg::kNPN)))
      bulk_in(s_npn, p.npn + (unit0 + p.chunks - 1 - d) * (Cfg::kNPN / 2), Cfg::kNPN, &full_n);
    }
    __syncwarp();
  };
  if (loads) {
    for (int64_t d = 0; d < min((int64_t)Cfg::kSt, p.chunks); ++d) load_kq(d);
    load_n(0);
  }

  const int64_t row0 = (b * p.L + tok) * vstride + (int64_t)h * p.dv + dv0;  // of token 0's chunk
  NextRow<T, C> next_do(sm0 + Cfg::oRow, (warp >> 2) * 64 + tok);
  auto load_do = [&](int64_t c) {
    next_do.fetch(static_cast<const T*>(p.grad) + row0 + c * kChunk * vstride,
                  c * kChunk + tok < p.L ? nval : 0, static_cast<const T*>(p.grad) FPSCAN_DEBUG_ONLY(, n_v));
  };
  if (!is_y) load_do(p.chunks - 1);

  float S[C];  // dS, one row of dk
#pragma unroll
  for (int i = 0; i < C; ++i)
    S[i] = p.grad_final != nullptr && dk < p.dk && i < nval FPSCAN_DEBUG_ONLY(
               && within<float, 4>(p.grad_final + (bh * p.dv + dv0 + i) * p.dk + dk, 1, p.grad_final, n_state))
               ? p.grad_final[(bh * p.dv + dv0 + i) * p.dk + dk]
               : 0.f;
  const int ksteps = (p.dk + 15) / 16;

  // Parts of a row of 32 values: to a stacked operand's row, to strips.
  auto put_tile = [&](int row, const float (&x)[C]) {
    split_row<NS>(x, [&](int q, int u, const uint4& w) {
      sts128(val_at<C>(s_e + q * Cfg::kPart, row, col0 / 8 + u), w);
    });
  };
  auto strip_ptr = [&](__nv_bfloat16* base, int64_t c, int u, int parts, int q, int bytes) {
    return reinterpret_cast<char*>(base) +
           (((unit0 + c) * strips + dv0 / 16 + (u >> 1)) * parts + q) * (int64_t)bytes;
  };

  bool ok = true;  // as in delta_scan_kernel
  auto wait = [&](uint64_t* bar, int64_t phase) {
    if (ok) ok = mbar_wait_soon(bar, (uint32_t)(phase & 1));
  };
  for (int64_t d = 0; d < p.chunks; ++d) {
    const int64_t c = p.chunks - 1 - d;
    const int s = (int)(d % Cfg::kSt);
    const uint32_t s_kq = sm0 + s * Cfg::kKQ;
    const float* vec = reinterpret_cast<const float*>(dsm + Cfg::oVec + s * Cfg::kVec);

    // dS's parts, rows of dk
    split_row<NS>(S, [&](int q, int u, const uint4& w) {
      sts128(val_at<C>(s_s + q * Cfg::kPart, dk, col0 / 8 + u), w);
    });
    fence_async();
    umma_fence_before();
    __syncthreads();
    if (loads && d > 0 && d + Cfg::kSt - 1 < p.chunks) load_kq(d + Cfg::kSt - 1);
    if (warp == 0) {
      umma_fence_after();
      wait(&full_kq[s], d / Cfg::kSt);
      if (elect_one()) {
        umma_parts<C, NP, LV, 8, true, false>(tmem, umma_desc_a(s_kq, 16), umma_desc_b<C>(s_s, Cfg::kPart),
                                              kTileKQ, 32, 64 * C, kHalfTile, ksteps);
        umma_commit(&done[0]);
      }
      __syncwarp();
    }
    // dS's parts to their strips, from the registers, while the product runs
    split_row<NS>(S, [&](int q, int u, const uint4& w) {
      if ((u & ~1) * 8 < nval FPSCAN_DEBUG_ONLY(
                                  && within<char>(strip_ptr(p.ds_parts, c, u, NS, q, 2 * kStrip) + strip_at(0, dk, u & 1), 16,
                                                  p.ds_parts, n_units * strips * NS * 2 * kStrip)))
        *reinterpret_cast<uint4*>(strip_ptr(p.ds_parts, c, u, NS, q, 2 * kStrip) + strip_at(0, dk, u & 1)) = w;
    });
    wait(&full_kq[s], d / Cfg::kSt);  // the vectors
    const float ge = vec[kVecEnter * kChunk + tok], total = vec[kVecEnter * kChunk + kChunk - 1];
    const float wb = vec[kVecLeave * kChunk + tok] * vec[kVecBeta * kChunk + tok];

    float x[C], g[C];
    if (!is_y) {
      next_do.take(g);
      split_row<NP>(g, [&](int q, int u, const uint4& w) {
        if ((u & ~1) * 8 < nval FPSCAN_DEBUG_ONLY(
                                    && within<char>(strip_ptr(p.do_parts, c, u, NP, q, kStrip) + strip_at(0, tok, u & 1), 16,
                                                    p.do_parts, n_units * strips * NP * kStrip)))
          *reinterpret_cast<uint4*>(strip_ptr(p.do_parts, c, u, NP, q, kStrip) +
                                    strip_at(0, tok, u & 1)) = w;
      });
      if (!Cfg::kOver) put_tile(kChunk + tok, g);
      if (c > 0) load_do(c - 1);
    }
    wait(&done[0], d);
    umma_fence_after();
    if (is_y) {
      tmem_sum<NS>(my_tmem, x);
#pragma unroll
      for (int i = 0; i < C; ++i) x[i] *= wb;
      put_tile(tok, x);
    } else if (Cfg::kOver) {
      put_tile(kChunk + tok, g);
    }
    fence_async();
    umma_fence_before();
    __syncthreads();
    if (warp == 0) {
      umma_fence_after();
      wait(&full_n, d);
      if (elect_one()) {
        umma_parts<C, NS, LV, 8, false, true>(tmem2, umma_desc_a(s_npn, 0), umma_desc_b<C>(s_e, Cfg::kPart),
                                              2 * kMatBytes, 2048, 64 * C, 0, 8);
        umma_commit(&done[1]);
      }
      __syncwarp();
    }
    wait(&done[1], d);
    umma_fence_after();
    if (loads && d + 1 < p.chunks) load_n(d + 1);  // N and PN are used up

    tmem_sum<NS>(my_tmem + NS * 2 * C, x);  // dV, in both halves of the lanes
    if (is_y) {
#pragma unroll
      for (int i = 0; i < C; ++i) g[i] = x[i] * -ge;
      put_tile(tok, g);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) g[i] *= ge * p.scale;
      put_tile(kChunk + tok, g);
    }
    fence_async();
    umma_fence_before();
    __syncthreads();
    if (warp == 0) {
      umma_fence_after();
      if (elect_one()) {
        umma_parts<C, NP, LV, 8, false, true>(tmem, umma_desc_a(s_kq, kHalfTile),
                                              umma_desc_b<C>(s_e, Cfg::kPart), kTileKQ, 2048, 64 * C, 0, 8);
        umma_commit(&done[2]);
      }
      __syncwarp();
    }
    // meanwhile: dV to the caller and as parts
    if (is_y) {
      split_row<NS>(x, [&](int q, int u, const uint4& w) {
        if ((u & ~1) * 8 < nval FPSCAN_DEBUG_ONLY(
                                    && within<char>(strip_ptr(p.dv_parts, c, u, NS, q, kStrip) + strip_at(0, tok, u & 1), 16,
                                                    p.dv_parts, n_units * strips * NS * kStrip)))
          *reinterpret_cast<uint4*>(strip_ptr(p.dv_parts, c, u, NS, q, kStrip) +
                                    strip_at(0, tok, u & 1)) = w;
      });
    } else if (c * kChunk + tok < p.L) {
      store_row<T>(static_cast<T*>(p.dv_out) + row0 + c * kChunk * vstride, nval,
                   x FPSCAN_DEBUG_ONLY(, p.dv_out, n_v));
    }
    wait(&done[2], d);
    umma_fence_after();
    tmem_sum<NS>(my_tmem, x);
#pragma unroll
    for (int i = 0; i < C; ++i) S[i] = fmaf(total, S[i], x[i]);
  }

  if (p.dinitial != nullptr && ok && dk < p.dk)
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (i < nval FPSCAN_DEBUG_ONLY(
                       && within<float, 4>(p.dinitial + (bh * p.dv + dv0 + i) * p.dk + dk, 1, p.dinitial, n_state)))
        p.dinitial[(bh * p.dv + dv0 + i) * p.dk + dk] = S[i];
  // No copy may land after the CTA is gone: at once, unless a wait gave up.
  if (loads) {
    for (int64_t d = max((int64_t)0, p.chunks - Cfg::kSt); d < p.chunks; ++d)
      mbar_wait_soon(&full_kq[d % Cfg::kSt], (uint32_t)((d / Cfg::kSt) & 1));
    mbar_wait_soon(&full_n, (uint32_t)((p.chunks - 1) & 1));
  }
  umma_fence_before();
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem));
}

// ------------------------------------------------------------------ gradients of a chunk
struct GradParams {
  const __nv_bfloat16* kq_tiles;
  const __nv_bfloat16* do_parts;
  const __nv_bfloat16* e_parts;
  const __nv_bfloat16* dv_parts;
  const __nv_bfloat16* s_parts;
  const __nv_bfloat16* ds_parts;
  const float* vecs;
  const void* log_decay;
  void* dq;              // T (batch, seqlen, key_heads, dk), or nullptr:
  void* dk_out;
  float* dq_part;        // fp32 (batch, seqlen, heads, dk), summed afterwards
  float* dk_part;
  void* dlog_decay;
  void* dbeta;
  int64_t L, chunks, units;  // units: chunks of all heads
  int key_heads, heads, dk, dv;
  float scale;
  int64_t nb;  // sequences (bounds checks of debug builds)
};

#ifdef FPSCAN_DEBUG_BOUNDS
// A strip of every kept tensor, K's and Q's tile and the vectors of a unit,
// inside what the call keeps.
template <int NP, int NS>
__device__ __forceinline__ bool strip_within(const GradParams& p, int64_t strip, int strips) {
  const int64_t n = p.units * strips;
  return within<char>(p.do_parts + strip * (NP * kStrip / 2), NP * kStrip, p.do_parts, n * NP * kStrip) &&
         within<char>(p.dv_parts + strip * (NS * kStrip / 2), NS * kStrip, p.dv_parts, n * NS * kStrip) &&
         within<char>(p.e_parts + strip * (NS * kStrip / 2), NS * kStrip, p.e_parts, n * NS * kStrip) &&
         within<char>(p.s_parts + strip * (NS * kStrip), NS * 2 * kStrip, p.s_parts, n * NS * 2 * kStrip) &&
         within<char>(p.ds_parts + strip * (NS * kStrip), NS * 2 * kStrip, p.ds_parts, n * NS * 2 * kStrip);
}
// N elements of dq, dk (`at`) or of their parts (`part`); an element of the decays and their gradients.
template <typename T, int N>
__device__ __forceinline__ bool grads_within(const GradParams& p, int64_t part, int64_t at) {
  const int64_t n = p.nb * p.L * p.dk;
  if (p.dq_part != nullptr)
    return within<float, 4 * N>(p.dq_part + part, N, p.dq_part, n * p.heads) &&
           within<float, 4 * N>(p.dk_part + part, N, p.dk_part, n * p.heads);
  return within<T, sizeof(T) * N>(static_cast<T*>(p.dq) + at, N, p.dq, n * p.key_heads) &&
         within<T, sizeof(T) * N>(static_cast<T*>(p.dk_out) + at, N, p.dk_out, n * p.key_heads);
}
template <typename T>
__device__ __forceinline__ bool decays_within(const GradParams& p, int64_t at) {
  const int64_t n = p.nb * p.L * p.heads;
  return within<T, sizeof(T)>(static_cast<const T*>(p.log_decay) + at, 1, p.log_decay, n) &&
         within<T, sizeof(T)>(static_cast<T*>(p.dlog_decay) + at, 1, p.dlog_decay, n) &&
         within<T, sizeof(T)>(static_cast<T*>(p.dbeta) + at, 1, p.dbeta, n);
}
template <int NP>
__device__ __forceinline__ bool tile_within(const GradParams& p, int64_t tile) {
  return within<char>(p.kq_tiles + tile, NP * kTileKQ, p.kq_tiles, p.nb * p.key_heads * p.chunks * NP * kTileKQ);
}
__device__ __forceinline__ bool vecs_within(const GradParams& p, int64_t unit) {
  return within<float>(p.vecs + unit * (kVecCount * kChunk), kVecCount * kChunk, p.vecs,
                       p.units * (kVecCount * kChunk));
}
#endif

constexpr int kGradThreads = 512;

// For 32-bit results (LV = 2; the sums of each step of 16 values have to be
// rounded, see Step, which products summed in tensor memory are not).  16
// warps.  The three 64 x dk sums (dQ, R, W) are cut into tiles of 32 rows x 16
// columns, H and X into tiles of 16 x 16; all stay in registers while dO, dV,
// E, S0 and dS pass once through a ring of bulk copies, a strip of 16 values
// at a time.  One CTA per SM takes chunk after chunk, and the ring runs on
// into the next chunk during the second phase.  Bound by mma.sync and its
// loads from shared memory (4 x 4096 tokens of 16 heads took its form for 16
// bits 542 us); 2 x 200 tokens of 4 heads, dk = dv = 64, fp32: 34 us (30 us
// with the sums that cancel in dlog_decay).
template <int NP>
struct GradCfg {
  static constexpr int LV = 2, NS = LV + 1;
  static constexpr int MT = 2;     // m tiles of a warp in the 64 x dk sums
  static constexpr int kColW = 8;  // warps side by side there
  static constexpr int kMat = kMatBytes;
  static constexpr int kRows = 2 * kStrip;  // a strip of a part of S0 or dS
  // a stage of the ring
  static constexpr int oV = NP * kStrip, oE = oV + NS * kStrip, oS = oE + NS * kStrip;
  static constexpr int oD = oS + NS * kRows, kStage = oD + NS * kRows;
  // K, Q and the decay vectors; two matrices of the second phase; the ring
  static constexpr int oVec = NP * kTileKQ;
  static constexpr int kVecBytes = kVecCount * kChunk * 4;
  static constexpr int oMats = oVec + (kVecBytes + 127) / 128 * 128;
  static constexpr int oRing = oMats + 2 * NS * kMat;
  static constexpr int kRoom = 227 * 1024 - 8192 - 128 - oRing;
  static constexpr int kStages = kRoom / kStage < 4 ? kRoom / kStage : 4;
  static constexpr int kSmem = oRing + kStages * kStage + 128;
  static_assert(kStages >= 1 && kSmem + 8192 <= 227 * 1024);
};

// sum_{i >= t} reads_i + sum_{j < t} writes_j for t = 2 lane, 2 lane + 1, of
// which the lane holds the values.
__device__ __forceinline__ void crossing_sums(const double (&reads)[2], const double (&writes)[2], int lane,
                                              double (&out)[2]) {
  double suffix = reads[0] + reads[1], prefix = writes[0] + writes[1];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double r = __shfl_down_sync(0xffffffffu, suffix, d);
    if (lane + d < 32) suffix += r;
    const double w = __shfl_up_sync(0xffffffffu, prefix, d);
    if (lane >= d) prefix += w;
  }
  // (lane by lane: a difference would let in what does not cross t)
  double behind = __shfl_down_sync(0xffffffffu, suffix, 1), before = __shfl_up_sync(0xffffffffu, prefix, 1);
  if (lane == 31) behind = 0.0;
  if (lane == 0) before = 0.0;
  out[0] = suffix + before;
  out[1] = (reads[1] + behind) + (before + writes[0]);
}

constexpr int kPadA = kChunk + 4;  // fp32 rows of A in shared memory: columns of eight rows on distinct banks

template <typename T>
__global__ void __launch_bounds__(kGradThreads, 1) delta_grad_kernel(const GradParams p) {
  constexpr int NP = kParts<T>;
  using Cfg = GradCfg<NP>;
  constexpr int LV = Cfg::LV, NS = Cfg::NS, NTH = kGradThreads, MROW = kChunk * 2;
  constexpr int MT = Cfg::MT, ST = Cfg::kStages, CW = Cfg::kColW;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t st = smem_addr(dsm);
  __shared__ float s_red[3][CW][kChunk];  // reads, k.W and writes / beta, by warp columns
  __shared__ float s_dot[NTH / 32], s_cross[kChunk];
  __shared__ __align__(8) uint64_t full[ST], freed[ST], full_kq;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int row0 = warp / CW * 16 * MT, col0 = warp % CW * 16;  // in the 64 x dk sums
  const int hr = (warp >> 2) * 16, hc = (warp & 3) * 16;        // in H and X
  // The tiles of H and X above the diagonal are not needed: their 6 warps
  // take <S0, dS> instead, and one thread of them (kLoader) issues the copies
  // (a whole warp with an elected lane spilled more: 29 us against 26 at 2 x 200 tokens).
  const bool lower = hc <= hr;
  constexpr int kLoader = 3 * 32;
  const int above = warp < 4 ? warp - 1 : warp < 8 ? warp - 3 : 5;  // 0..5 among those
  const int64_t kstride = (int64_t)p.key_heads * p.dk;
  const int strips = (p.dv + 15) / 16;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&freed[i], NTH / 32);
    }
    mbar_init(&full_kq, 1);
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // the copies: strip by strip, over this CTA's chunks
  const int64_t mine = (p.units - blockIdx.x + gridDim.x - 1) / gridDim.x;  // chunks of this CTA
  const int64_t total = mine * strips;
  int64_t next = 0;      // strips issued
  int64_t next_unit = blockIdx.x;
  int next_strip = 0;
  auto issue = [&]() {
    const int s = (int)(next % ST);
    if (next >= ST && !mbar_wait_soon(&freed[s], (uint32_t)((next / ST - 1) & 1))) return;
    const int64_t strip = next_unit * strips + next_strip;
    const uint32_t at = st + Cfg::oRing + s * Cfg::kStage;
    mbar_expect_tx(&full[s], Cfg::kStage);
    FPSCAN_DEBUG_ONLY(if (strip_within<NP, NS>(p, strip, strips)) {)
    bulk_in(at, p.do_parts + strip * (NP * kStrip / 2), NP * kStrip, &full[s]);
    bulk_in(at + Cfg::oV, p.dv_parts + strip * (NS * kStrip / 2), NS * kStrip, &full[s]);
    bulk_in(at + Cfg::oE, p.e_parts + strip * (NS * kStrip / 2), NS * kStrip, &full[s]);
    bulk_in(at + Cfg::oS, p.s_parts + strip * (NS * Cfg::kRows / 2), NS * Cfg::kRows, &full[s]);
    bulk_in(at + Cfg::oD, p.ds_parts + strip * (NS * Cfg::kRows / 2), NS * Cfg::kRows, &full[s]);
    FPSCAN_DEBUG_ONLY(})
    ++next;
    if (++next_strip == strips) {
      next_strip = 0;
      next_unit += gridDim.x;
    }
  };
  auto issue_kq = [&](int64_t unit) {
    const int64_t bh = unit / p.chunks, chunk = unit - bh * p.chunks, b = bh / p.heads;
    const int hk = (int)(bh - b * p.heads) / (p.heads / p.key_heads);
    const int64_t tile = ((b * p.key_heads + hk) * p.chunks + chunk) * NP * (kTileKQ / 2);
    mbar_expect_tx(&full_kq, NP * kTileKQ + Cfg::kVecBytes);
    FPSCAN_DEBUG_ONLY(if (!tile_within<NP>(p, tile) || !vecs_within(p, unit)) return;)
    bulk_in(st, p.kq_tiles + tile, NP * kTileKQ, &full_kq);
    bulk_in(st + Cfg::oVec, p.vecs + unit * (kVecCount * kChunk), Cfg::kVecBytes, &full_kq);
  };
  if (tid == kLoader) {
    const int64_t ahead = min((int64_t)ST, total);
    for (int64_t i = 0; i < ahead; ++i) issue();
    issue_kq(blockIdx.x);
  }

  bool ok = true;
  int64_t it = 0;  // strips consumed
  for (int64_t done = 0; done < mine; ++done) {
    const int64_t unit = blockIdx.x + done * gridDim.x;
    const int64_t bh = unit / p.chunks, chunk = unit - bh * p.chunks, b = bh / p.heads;
    const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
    const int64_t t0 = chunk * kChunk;
    const int rows = (int)min((int64_t)kChunk, p.L - t0);

    float aq[MT][2][4], ar[MT][2][4], aw[MT][2][4], ah[2][4], ax[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int m = 0; m < MT; ++m) aq[m][n][e] = ar[m][n][e] = aw[m][n][e] = 0.f;
        ah[n][e] = ax[n][e] = 0.f;
      }
    float dot = 0.f;  // this thread's share of <S0, dS>

    for (int sl = 0; sl < strips; ++sl, ++it) {
      const int s_id = (int)(it % ST);
      const uint32_t at = st + Cfg::oRing + s_id * Cfg::kStage;
      // refill the stage of the strip before: every warp is done with it, or nearly
      if (tid == kLoader && ST > 1 && it > 0 && next < total) issue();
      ok = __all_sync(0xffffffffu, mbar_wait_soon(&full[s_id], (uint32_t)((it / ST) & 1)));
      if (!ok) break;
      {
        const uint32_t a_v = at + Cfg::oV, a_e = at + Cfg::oE;
        if (lower) {
          uint32_t ag[NP][4], av[NS][4];
#pragma unroll
          for (int i = 0; i < NP; ++i) ldsm4(ag[i], strip_a(at + i * kStrip, lane, hr));
#pragma unroll
          for (int i = 0; i < NS; ++i) ldsm4(av[i], strip_a(a_v + i * kStrip, lane, hr));
          Step<true, 4> s;
#pragma unroll
          for (int j = LV; j >= 0; --j) {
            uint32_t eb[4];
            ldsm4(eb, strip_b(a_e + j * kStrip, lane, hc));
#pragma unroll
            for (int i = LV - j; i >= 0; --i) {
              if (i < NP) {
                s.mma(0, ah[0], ag[i < NP ? i : 0], eb[0], eb[1]);
                s.mma(1, ah[1], ag[i < NP ? i : 0], eb[2], eb[3]);
              }
              s.mma(2, ax[0], av[i], eb[0], eb[1]);
              s.mma(3, ax[1], av[i], eb[2], eb[3]);
            }
          }
          s.add(0, ah[0]);
          s.add(1, ah[1]);
          s.add(2, ax[0]);
          s.add(3, ax[1]);
        }
        {
          uint32_t sb[NS][4];
#pragma unroll
          for (int j = 0; j < NS; ++j)
            ldsm4(sb[j], strip_b(at + Cfg::oS + j * Cfg::kRows, lane, col0));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            uint32_t ag[NP][4], av[NS][4];
#pragma unroll
            for (int i = 0; i < NP; ++i) ldsm4(ag[i], strip_a(at + i * kStrip, lane, row0 + m * 16));
#pragma unroll
            for (int i = 0; i < NS; ++i) ldsm4(av[i], strip_a(a_v + i * kStrip, lane, row0 + m * 16));
            Step<true, 4> s;
#pragma unroll
            for (int j = LV; j >= 0; --j)
#pragma unroll
              for (int i = LV - j; i >= 0; --i) {
                if (i < NP) {
                  s.mma(0, aq[m][0], ag[i < NP ? i : 0], sb[j][0], sb[j][1]);
                  s.mma(1, aq[m][1], ag[i < NP ? i : 0], sb[j][2], sb[j][3]);
                }
                s.mma(2, ar[m][0], av[i], sb[j][0], sb[j][1]);
                s.mma(3, ar[m][1], av[i], sb[j][2], sb[j][3]);
              }
            s.add(0, aq[m][0]);
            s.add(1, aq[m][1]);
            s.add(2, ar[m][0]);
            s.add(3, ar[m][1]);
          }
        }
        {
          uint32_t db[NS][4];
#pragma unroll
          for (int j = 0; j < NS; ++j)
            ldsm4(db[j], strip_b(at + Cfg::oD + j * Cfg::kRows, lane, col0));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            uint32_t ae[NS][4];
#pragma unroll
            for (int i = 0; i < NS; ++i) ldsm4(ae[i], strip_a(a_e + i * kStrip, lane, row0 + m * 16));
            Step<true, 2> s;
#pragma unroll
            for (int j = LV; j >= 0; --j)
#pragma unroll
              for (int i = LV - j; i >= 0; --i) {
                s.mma(0, aw[m][0], ae[i], db[j][0], db[j][1]);
                s.mma(1, aw[m][1], ae[i], db[j][2], db[j][3]);
              }
            s.add(0, aw[m][0]);
            s.add(1, aw[m][1]);
          }
        }
      }
      // <S0, dS> over this strip (the same place of every part: swizzle does not matter)
      for (int i = above * 32 + lane; !lower && i < Cfg::kRows / 16; i += 6 * 32) {
        float x[8] = {}, y[8] = {};
#pragma unroll
        for (int q = NS - 1; q >= 0; --q) {
          const uint4 u = lds128(at + Cfg::oS + q * Cfg::kRows + i * 16);
          const uint4 v = lds128(at + Cfg::oD + q * Cfg::kRows + i * 16);
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[2 * e] += bf16_lo(uw[e]);
            x[2 * e + 1] += bf16_hi(uw[e]);
            y[2 * e] += bf16_lo(vw[e]);
            y[2 * e + 1] += bf16_hi(vw[e]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(x[e], y[e], dot);
      }
      warp_arrive(&freed[s_id], lane);
      if (tid == kLoader && ST == 1 && next < total) issue();
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (lane == 0) s_dot[warp] = dot;
    ok = ok && mbar_wait_soon(&full_kq, (uint32_t)(done & 1));
    if (__syncthreads_or(!ok)) {
      ok = false;
      break;
    }

    // second phase
    const float* s_vec = reinterpret_cast<const float*>(dsm + Cfg::oVec);
    const float* enter = s_vec + kVecEnter * kChunk;
    const float* leave = s_vec + kVecLeave * kChunk;
    const float* beta = s_vec + kVecBeta * kChunk;
    const float* hi = s_vec + kVecCumHi * kChunk;
    const float* lo = s_vec + kVecCumLo * kChunk;
    // H and X times D: rows i, columns j, in the order of an A operand's
    // registers.  As parts in shared memory first with each column times beta
    // (set 0, row operands of dQ and R), then without (set 1, column operands
    // of W).
    float2 hd[4], xd[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = q >> 1, r = q & 1;
      const int i = hr + r * 8 + g4, j0 = hc + n * 8 + 2 * t4;
      hd[q] = xd[q] = make_float2(0.f, 0.f);
      if (lower) {
        const float2 hj = *reinterpret_cast<const float2*>(hi + j0);
        const float2 lj = *reinterpret_cast<const float2*>(lo + j0);
        const float d0 = i > j0 ? expf((hi[i] - hj.x) + (lo[i] - lj.x)) : 1.f;
        const float d1 = i > j0 + 1 ? expf((hi[i] - hj.y) + (lo[i] - lj.y)) : 1.f;
        if (i >= j0) hd[q].x = ah[n][2 * r] * d0 * p.scale;
        if (i >= j0 + 1) hd[q].y = ah[n][2 * r + 1] * d1 * p.scale;
        if (i > j0) xd[q].x = -ax[n][2 * r] * d0;
        if (i > j0 + 1) xd[q].y = -ax[n][2 * r + 1] * d1;
      }
    }
    auto put_mats = [&](int set) {
      const uint32_t base = st + Cfg::oMats;
      uint32_t wh[4][NS], wx[4][NS];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float2 w = make_float2(1.f, 1.f);
        if (set == 0) w = *reinterpret_cast<const float2*>(beta + hc + (q >> 1) * 8 + 2 * t4);
        split_pair<NS>(hd[q].x * w.x, hd[q].y * w.y, wh[q]);
        split_pair<NS>(xd[q].x * w.x, xd[q].y * w.y, wx[q]);
      }
#pragma unroll
      for (int q = 0; q < NS; ++q) {
        const uint32_t a[4] = {wh[0][q], wh[1][q], wh[2][q], wh[3][q]};
        const uint32_t x[4] = {wx[0][q], wx[1][q], wx[2][q], wx[3][q]};
        stsm4(at_a<MROW>(base + q * Cfg::kMat, lane, hr, hc / 16), a);
        stsm4(at_a<MROW>(base + (NS + q) * Cfg::kMat, lane, hr, hc / 16), x);
      }
    };
    // an element pair of K or Q as fp32 (the sum of its parts)
    auto kq_pair = [&](int row, int col) {  // Q: rows 64..
      float2 v = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = NP - 1; i >= 0; --i) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(
            dsm + i * kTileKQ + (col >> 6) * kHalfTile + tile_at<128>(0, row, (col & 63) / 8) +
            (col % 8) * 2);
        v.x += bf16_lo(w);
        v.y += bf16_hi(w);
      }
      return v;
    };
    // this warp's columns of K (and, 64 rows on, Q) as a B operand
    const uint32_t kq_cols = st + (col0 >> 6) * kHalfTile;
    // A, the sum of its rows up to each t, and of those over i >= t (in the
    // room of the matrices).  The tokens' products are made here a second time:
    // the first were for the forward pass, in another kernel.
    float* s_a = reinterpret_cast<float*>(dsm + Cfg::oMats);
    {
      float2 z[4] = {};
      if (lower) {
        const int ksteps = (p.dk + 15) / 16;
#pragma unroll
        for (int which = 0; which < 2; ++which) {  // K K^T, Q K^T
          float t[2][4] = {};
          for (int kk = 0; kk < ksteps; ++kk) {
            const uint32_t half = st + (kk >> 2) * kHalfTile;
            Step<true, 2> sum;
#pragma unroll
            for (int j = NP - 1; j >= 0; --j) {
              uint32_t kb[4];
              ldsm4(kb, at_b<128>(half + j * kTileKQ, lane, hc, kk & 3));
#pragma unroll
              for (int i = NP - 1; i >= 0; --i) {
                if (i + j > LV) continue;
                uint32_t a[4];
                ldsm4(a, at_a<128>(half + i * kTileKQ, lane, which * kChunk + hr, kk & 3));
                sum.mma(0, t[0], a, kb[0], kb[1]);
                sum.mma(1, t[1], a, kb[2], kb[3]);
              }
            }
            sum.add(0, t[0]);
            sum.add(1, t[1]);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 f = which ? hd[q] : xd[q];
            z[q].x = fmaf(f.x, t[q >> 1][2 * (q & 1)], z[q].x);
            z[q].y = fmaf(f.y, t[q >> 1][2 * (q & 1) + 1], z[q].y);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = hr + (q & 1) * 8 + g4, j0 = hc + (q >> 1) * 8 + 2 * t4;
        const float2 w = *reinterpret_cast<const float2*>(beta + j0);
        *reinterpret_cast<float2*>(&s_a[i * kPadA + j0]) =
            make_float2(i > j0 ? z[q].x * w.x : 0.f, i > j0 + 1 ? z[q].y * w.y : 0.f);
      }
      __syncthreads();
      const int i = tid >> 3, part = tid & 7;  // a row, eight of its columns
      float a[8], sum = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float v = s_a[i * kPadA + part * 8 + c];
        a[c] = sum;
        sum += v;
      }
      float left = sum;
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) {
        const float o = __shfl_up_sync(0xffffffffu, left, d, 8);
        if (part >= d) left += o;
      }
      left = __shfl_up_sync(0xffffffffu, left, 1, 8);
      if (part == 0) left = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        s_a[i * kPadA + part * 8 + c] = part * 8 + c <= i ? left + a[c] : 0.f;
      __syncthreads();
      float cross = 0.f;  // t = i: rows part, part + 8, ..
#pragma unroll
      for (int c = 0; c < 8; ++c) cross += s_a[(part + 8 * c) * kPadA + i];
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) cross += __shfl_xor_sync(0xffffffffu, cross, d);
      if (part == 0) s_cross[i] = cross;
      __syncthreads();
    }
    put_mats(0);
    // sums over a warp's columns of a row, one value per row and warp column
    auto put_row = [&](int which, int row, float v) {
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (t4 == 0) s_red[which][warp % CW][row] = v;
    };
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = row0 + m * 16 + r * 8 + g4;
        const float ge = enter[i], gl = leave[i];
        float reads = 0.f, writes = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float2 kv = kq_pair(i, col0 + n * 8 + 2 * t4);
          const float2 qv = kq_pair(kChunk + i, col0 + n * 8 + 2 * t4);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            aq[m][n][2 * r + c] *= ge * p.scale;
            ar[m][n][2 * r + c] *= -ge;
            aw[m][n][2 * r + c] *= gl;
            reads = fmaf(aq[m][n][2 * r + c], c ? qv.y : qv.x, reads);
            reads = fmaf(ar[m][n][2 * r + c], c ? kv.y : kv.x, reads);
            writes = fmaf(aw[m][n][2 * r + c], c ? kv.y : kv.x, writes);
          }
        }
        put_row(0, i, reads);
        put_row(2, i, writes);
      }
    __syncthreads();

    // dQ += Hb K, R += Xb K: rows i, columns j <= i
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk * 16 > row0 + 16 * MT - 1) break;
      uint32_t kb[NP][4];
#pragma unroll
      for (int j = 0; j < NP; ++j) ldsm4_t(kb[j], at_bt<128>(kq_cols + j * kTileKQ, lane, col0 & 63, kk));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Step<true, 4> s;
#pragma unroll
        for (int i = LV; i >= 0; --i) {
          uint32_t fh[4], fx[4];
          const uint32_t base = st + Cfg::oMats + i * Cfg::kMat;
          ldsm4(fh, at_a<MROW>(base, lane, row0 + m * 16, kk));
          ldsm4(fx, at_a<MROW>(base + NS * Cfg::kMat, lane, row0 + m * 16, kk));
#pragma unroll
          for (int j = NP - 1; j >= 0; --j) {
            if (i + j > LV) continue;
            s.mma(0, aq[m][0], fh, kb[j][0], kb[j][1]);
            s.mma(1, aq[m][1], fh, kb[j][2], kb[j][3]);
            s.mma(2, ar[m][0], fx, kb[j][0], kb[j][1]);
            s.mma(3, ar[m][1], fx, kb[j][2], kb[j][3]);
          }
        }
        s.add(0, aq[m][0]);
        s.add(1, aq[m][1]);
        s.add(2, ar[m][0]);
        s.add(3, ar[m][1]);
      }
    }
    __syncthreads();
    put_mats(1);
    __syncthreads();
    // W += Hs^T Q + Xd^T K: rows j, columns i >= j
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk * 16 + 15 < row0) continue;
      uint32_t kb[NP][4], qb[NP][4];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        ldsm4_t(kb[j], at_bt<128>(kq_cols + j * kTileKQ, lane, col0 & 63, kk));
        ldsm4_t(qb[j], at_bt<128>(kq_cols + j * kTileKQ + kChunk * 128, lane, col0 & 63, kk));
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Step<true, 4> s;
#pragma unroll
        for (int i = LV; i >= 0; --i) {
          uint32_t fh[4], fx[4];
          const uint32_t base = st + Cfg::oMats + i * Cfg::kMat;
          ldsm4_t(fh, at_at<MROW>(base, lane, row0 + m * 16, kk));
          ldsm4_t(fx, at_at<MROW>(base + NS * Cfg::kMat, lane, row0 + m * 16, kk));
#pragma unroll
          for (int j = NP - 1; j >= 0; --j) {
            if (i + j > LV) continue;
            s.mma(0, aw[m][0], fh, qb[j][0], qb[j][1]);
            s.mma(1, aw[m][1], fh, qb[j][2], qb[j][3]);
            s.mma(2, aw[m][0], fx, kb[j][0], kb[j][1]);
            s.mma(3, aw[m][1], fx, kb[j][2], kb[j][3]);
          }
        }
        s.add(0, aw[m][0]);
        s.add(1, aw[m][1]);
        s.add(2, aw[m][0]);
        s.add(3, aw[m][1]);
      }
    }

    const int64_t kf = (b * p.L + t0) * kstride + (int64_t)hk * p.dk;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = row0 + m * 16 + r * 8 + g4;
        const float be = beta[i];
        float kw = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int col = col0 + n * 8 + 2 * t4;
          const float2 kv = kq_pair(i, col);
          const float q0 = aq[m][n][2 * r], q1 = aq[m][n][2 * r + 1];
          const float r0 = ar[m][n][2 * r], r1 = ar[m][n][2 * r + 1];
          const float w0 = aw[m][n][2 * r], w1 = aw[m][n][2 * r + 1];
          kw = fmaf(kv.x, w0, fmaf(kv.y, w1, kw));
          const float k0 = fmaf(be, w0, r0), k1 = fmaf(be, w1, r1);
          if (i < rows && col < p.dk FPSCAN_DEBUG_ONLY(
                              && grads_within<T, 2>(p, ((b * p.L + t0 + i) * p.heads + h) * p.dk + col,
                                                    kf + (int64_t)i * kstride + col))) {
            if (p.dq_part != nullptr) {
              const int64_t o = ((b * p.L + t0 + i) * p.heads + h) * p.dk + col;
              *reinterpret_cast<float2*>(p.dq_part + o) = make_float2(q0, q1);
              *reinterpret_cast<float2*>(p.dk_part + o) = make_float2(k0, k1);
            } else {
              const int64_t o = kf + (int64_t)i * kstride + col;
              T* dq = static_cast<T*>(p.dq) + o;
              T* dk = static_cast<T*>(p.dk_out) + o;
              if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float2*>(dq) = make_float2(q0, q1);
                *reinterpret_cast<float2*>(dk) = make_float2(k0, k1);
              } else {
                *reinterpret_cast<uint32_t*>(dq) = pack2<T>(q0, q1);
                *reinterpret_cast<uint32_t*>(dk) = pack2<T>(k0, k1);
              }
            }
          }
        }
        put_row(1, i, kw);
      }
    __syncthreads();

    // dbeta, and the sums of dlog_decay: one warp, two tokens a lane, in 64 bits
    if (warp == 0) {
      double reads[2], writes[2], state = 0.0;
      float db[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 2 * lane + c;
        float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < CW; ++w)
#pragma unroll
          for (int q = 0; q < 3; ++q) sum[q] += s_red[q][w][i];
        reads[c] = sum[0];
        db[c] = sum[1];
        writes[c] = (double)beta[i] * (double)sum[2];
      }
      if (lane < NTH / 32) state = (double)enter[kChunk - 1] * (double)s_dot[lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) state += __shfl_xor_sync(0xffffffffu, state, d);
      double out[2];
      crossing_sums(reads, writes, lane, out);
#pragma unroll
      for (int c = 0; c < 2; ++c) out[c] += state + (double)s_cross[2 * lane + c];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 2 * lane + c;
        if (i < rows) {
          const int64_t o = (b * p.L + t0 + i) * p.heads + h;
          FPSCAN_DEBUG_ONLY(if (!decays_within<T>(p, o)) continue;)
          // a decay of exactly 0 has no slope in its logarithm
          const bool reset = Elem<T>::load(static_cast<const T*>(p.log_decay)[o]) < kDecayFloor;
          static_cast<T*>(p.dlog_decay)[o] = Elem<T>::store(reset ? 0.f : (float)out[c]);
          static_cast<T*>(p.dbeta)[o] = Elem<T>::store(db[c]);
        }
      }
    }
    __syncthreads();  // K, Q, the vectors and the sums are used up
    if (tid == kLoader && done + 1 < mine) issue_kq(unit + gridDim.x);
  }
  // After a wait that gave up: no copy may land after the CTA is gone.
  if (!ok && tid == kLoader) {
    for (int64_t j = max((int64_t)0, next - ST); j < next; ++j)
      mbar_wait_soon(&full[j % ST], (uint32_t)((j / ST) & 1));
    mbar_wait_soon(&full_kq, 0);
    mbar_wait_soon(&full_kq, 1);
  }
}

// ------------------------------------------------------------------ gradients of a chunk, tcgen05
// What delta_grad_kernel computes, for 16-bit results (LV = 1).  The sums are
// taken transposed, 128 rows of dk by 64 tokens, so that every product has
// 128 rows, and the strips are operands as they lie (32-byte rows and swizzle,
// 16 values of k each):
//     S0 [dV; dO]^T  -> R | dQ,   dS E^T -> W,   [dV; dO] E^T -> [X; H]
// strip by strip as they arrive, then
//     K^T [Xb; Hb]^T -> R | dQ,   [K; Q]^T [Xd; Hs] -> W
// with the matrices that the warps make of H and X, and [K; Q] K^T, which makes
// A of them.  20 warps: sixteen take the
// first sums into registers (the next chunk's first products may then start),
// make the matrices, add the second sums and write the gradients from there
// (a thread has one of dk and 16 tokens: 64 bytes a store, which costs less
// than turning the sums around through shared memory did); one issues all
// products, two take <S0, dS> from the strips as they pass (the first of them
// issues their copies), and one loads K, Q and the vectors and closes a chunk
// (dlog_decay, dbeta) behind the others.  Copies, like products, are issued by
// an elected lane of a converged warp: six copies took a lone thread of a
// divergent branch 900 cycles.  What bounds it: reading operands from shared
// memory, 640 KB a chunk at 128 bytes a cycle, and the warps' steps between
// the two phases.  4 x 4096 tokens of 16 heads, dk = dv = 128, bf16: 346 us
// (1.1 GB, 3.2 TB/s), 2 x 2048 with two value heads to a key head 91 us; A and
// what crosses each token cost 43 and 8 us of that over sums that cancel.
constexpr int kTcThreads = 640;  // 96 registers a thread; one warp more, and it is 80

template <int NP>
struct TcGradCfg {
  static constexpr int NS = 2;
  // a stage: parts p of [dV; dO] (dO's second part is zeros where NP = 1), E, S0, dS
  static constexpr int oE = 2 * 2 * kStrip, oS = oE + NS * kStrip, oD = oS + NS * 2 * kStrip;
  static constexpr int kStage = oD + NS * 2 * kStrip;
  static constexpr int kTx = (NP + 2 * NS) * kStrip + 2 * NS * 2 * kStrip;
  // K and Q; two matrices of two parts; the ring; decay vectors, those of the
  // next chunk too.  kStatic bytes besides (the kernel's __shared__ variables)
  static constexpr int kStatic = 11 * 1024 + 512;
  static constexpr int oM = NP * kTileKQ;
  static constexpr int kMatP = 128 * 128;  // a part of [Xb; Hb] or [Xd; Hs]
  static constexpr int oRing = oM + 2 * NS * kMatP;
  static constexpr int kVecBytes = kVecCount * kChunk * 4;
  static constexpr int kRoom = 227 * 1024 - 1024 - kStatic - 2 * kVecBytes;
  static constexpr int kStages = (kRoom - oRing) / kStage < 4 ? (kRoom - oRing) / kStage : 4;
  static constexpr int oVec = oRing + kStages * kStage;
  static constexpr int kSmem = oVec + 2 * kVecBytes + 1024;
  static_assert(kStages >= 2 && kSmem + kStatic <= 227 * 1024);
};

// K-major operand of strips: 32-byte rows and swizzle, 16 values of k.
__device__ __forceinline__ uint64_t umma_desc_strip(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t(1) << 16) | ((uint64_t)(256 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(6) << 61);
}
// Position in a ring of ST stages and how often it has gone round.
template <int ST>
struct Ring {
  int at = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == ST) {
      at = 0;
      ++phase;
    }
  }
};

// 16 values of every lane summed over each half of the warp: lane l keeps the
// sum of the values l & 15 of its half, in x[0].
__device__ __forceinline__ void over_lanes(float (&x)[16], int lane) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) {
#pragma unroll
    for (int c = 0; c < m; ++c) {
      const float send = lane & m ? x[c] : x[c + m], keep = lane & m ? x[c + m] : x[c];
      x[c] = keep + __shfl_xor_sync(0xffffffffu, send, m);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1) delta_grad_tc_kernel(const GradParams p) {
  constexpr int NP = kParts<T>;
  using Cfg = TcGradCfg<NP>;
  constexpr int NS = Cfg::NS, ST = Cfg::kStages;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t st = smem_addr(dsm);
  const uint32_t s_t1 = st + Cfg::oM, s_t2 = s_t1 + NS * Cfg::kMatP;
  __shared__ __align__(8) uint64_t full[ST], freed[ST], full_kq, full_vec[2], dots[2], done1, mats,
      done2, used_kq;
  __shared__ uint32_t s_tmem;
  // reads, writes / beta and k.W of every token, by quarters of dk; the sum of
  // A over its 16 columns from t & ~15 up to t and 32 rows i >= t
  __shared__ float s_rows[2][4][4][kChunk], s_dot[2][2];
  __shared__ float s_a[2][3][128];  // A's rows (X's share, H's share), summed over 16 columns

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform
  const int strips = (p.dv + 15) / 16;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&freed[i], 1 + 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full_vec[i], 1);
      mbar_init(&dots[i], 2);
    }
    mbar_init(&full_kq, 1);
    mbar_init(&done1, 1);
    mbar_init(&mats, 16);
    mbar_init(&done2, 1);
    mbar_init(&used_kq, 16);
    fence_mbar_init();
  }
  if (NP == 1)  // dO's second part
    for (int i = tid; i < ST * kStrip / 16; i += kTcThreads)
      sts128(st + Cfg::oRing + i / (kStrip / 16) * Cfg::kStage + 3 * kStrip + i % (kStrip / 16) * 16,
             make_uint4(0, 0, 0, 0));
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_addr(&s_tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_async();
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t t_w = tmem + 128, t_xh = tmem + 192, t_rq2 = tmem + 256, t_w2 = tmem + 384;
  const uint32_t t_kk = tmem + 448;
  pdl_wait();
  pdl_launch_dependents();

  const int64_t mine = (p.units - blockIdx.x + gridDim.x - 1) / gridDim.x;  // chunks of this CTA
  bool ok = true;  // as in delta_scan_kernel
  auto wait = [&](uint64_t* bar, int64_t phase) {
    if (ok) ok = mbar_wait_soon(bar, (uint32_t)(phase & 1));
  };

  if (warp == 16) {
    // ---------------------------------------------------------- products
    Ring<ST> ring;
    for (int64_t k = 0; k < mine; ++k) {
      for (int sl = 0; sl < strips; ++sl, ring.next()) {
        const int s = ring.at;
        wait(&full[s], ring.phase);
        umma_fence_after();
        __syncwarp();
        if (elect_one()) {
          const uint32_t at = st + Cfg::oRing + s * Cfg::kStage;
          const uint64_t dv = umma_desc_strip(at), e = umma_desc_strip(at + Cfg::oE),
                         s0 = umma_desc_strip(at + Cfg::oS), ds = umma_desc_strip(at + Cfg::oD);
          constexpr uint32_t pd = 2 * kStrip >> 4, pe = kStrip >> 4, ps = 2 * kStrip >> 4;  // parts
          const bool on = sl > 0;
          umma(tmem, s0 + ps, dv, umma_idesc(false, false, 128), on);
          umma(tmem, s0, dv + pd, umma_idesc(false, false, 128), true);
          umma(tmem, s0, dv, umma_idesc(false, false, 128), true);
          umma(t_w, ds + ps, e, umma_idesc(false, false, 64), on);
          umma(t_w, ds, e + pe, umma_idesc(false, false, 64), true);
          umma(t_w, ds, e, umma_idesc(false, false, 64), true);
          umma(t_xh, dv + pd, e, umma_idesc(false, false, 64), on);
          umma(t_xh, dv, e + pe, umma_idesc(false, false, 64), true);
          umma(t_xh, dv, e, umma_idesc(false, false, 64), true);
          umma_commit(&freed[s]);
          if (sl == strips - 1) umma_commit(&done1);
        }
        __syncwarp();
      }
      // (the warps were through with the chunk before's when K and Q were loaded)
      wait(&full_kq, k);
      umma_fence_after();
      __syncwarp();
      if (elect_one()) {
        const uint64_t kq = umma_desc_a(st, 16);
        bool on = false;
#pragma unroll
        for (int lv = 1; lv >= 0; --lv)
#pragma unroll
          for (int i = 0; i <= lv; ++i)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              if (i < NP && lv - i < NP) {
                const uint32_t at = (ks >> 2) * kHalfTile + (ks & 3) * 32;
                umma(t_kk, kq + ((i * kTileKQ + at) >> 4), kq + (((lv - i) * kTileKQ + at) >> 4),
                     umma_idesc(false, false, 64), on);
                on = true;
              }
      }
      __syncwarp();
      wait(&mats, k);
      umma_fence_after();
      __syncwarp();
      if (elect_one()) {
        const uint64_t kt = umma_desc_a(st, kHalfTile), t1 = umma_desc_a(s_t1, 16), t2 = umma_desc_a(s_t2, 16);
        bool on = false;
#pragma unroll
        for (int lv = 1; lv >= 0; --lv)
#pragma unroll
          for (int i = 0; i <= lv && i < NP; ++i)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              umma(t_rq2, kt + ((i * kTileKQ + ks * 2048) >> 4),
                   t1 + (((lv - i) * Cfg::kMatP + ks * 32) >> 4), umma_idesc(true, false, 128), on);
              on = true;
            }
        on = false;
#pragma unroll
        for (int lv = 1; lv >= 0; --lv)
#pragma unroll
          for (int i = 0; i <= lv && i < NP; ++i)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
              umma(t_w2, kt + ((i * kTileKQ + ks * 2048) >> 4),
                   t2 + (((lv - i) * Cfg::kMatP + ks * 2048) >> 4), umma_idesc(true, true, 64), on);
              on = true;
            }
        umma_commit(&done2);
      }
      __syncwarp();
    }
    // no product may run after the CTA is gone: at once, unless a wait gave up
    mbar_wait_soon(&done2, (uint32_t)((mine - 1) & 1));
  } else if (warp < 16) {
    // ---------------------------------------------------------- sums, matrices and rows
    const int quad = warp & 3, t0c = (warp >> 2) * 16;  // this thread's 16 columns
    const int row = quad * 32 + lane;  // lane of tensor memory: X, H row; row of dk
    const uint32_t my = ((uint32_t)(quad * 32) << 16) + t0c;
    const int64_t kstride = (int64_t)p.key_heads * p.dk, pstride = (int64_t)p.heads * p.dk;
    // this thread's row of dk of K (Q: rows from 64), as fp32 (the sum of its parts)
    auto kq1 = [&](int r) {
      float v = 0.f;
#pragma unroll
      for (int i = NP - 1; i >= 0; --i)
        v += __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(
            dsm + i * kTileKQ + (row >> 6) * kHalfTile + tile_at<128>(0, r, (row & 63) / 8) + (row % 8) * 2));
      return v;
    };
    for (int64_t k = 0; k < mine; ++k) {
      const int64_t unit = blockIdx.x + k * gridDim.x;
      const int64_t bh = unit / p.chunks, chunk = unit - bh * p.chunks, b = bh / p.heads;
      const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
      const int64_t t0 = chunk * kChunk;
      const int rows = (int)min((int64_t)kChunk, p.L - t0);
      const int buf = (int)(k & 1);
      const float* vec = reinterpret_cast<const float*>(dsm + Cfg::oVec + buf * Cfg::kVecBytes);
      const float* beta = vec + kVecBeta * kChunk;

      wait(&full_vec[buf], k >> 1);
      wait(&done1, k);
      umma_fence_after();
      auto vec16 = [&](int which, float (&v)[16]) {  // of this thread's columns
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 f = *reinterpret_cast<const float4*>(vec + which * kChunk + t0c + 4 * c);
          v[4 * c] = f.x;
          v[4 * c + 1] = f.y;
          v[4 * c + 2] = f.z;
          v[4 * c + 3] = f.w;
        }
      };
      float x[16], dq[16], r[16], w[16];
      {
        // X (rows 0..63) or H (64..127), row i, columns j: times D; with each
        // column times beta to [Xb; Hb], without to [Xd; Hs]
        tmem_ld(t_xh + my, x);
        const int i = row & 63;
        const bool is_h = row >= 64;
        const float hi_i = vec[kVecCumHi * kChunk + i], lo_i = vec[kVecCumLo * kChunk + i];
        const float f = is_h ? p.scale : -1.f;
        float hi[16], lo[16];
        vec16(kVecCumHi, hi);
        vec16(kVecCumLo, lo);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const int j = t0c + c;
          // (an error of 2^-16 of D at the most, where D is above e^-80)
          const float d = i > j ? __expf((hi_i - hi[c]) + (lo_i - lo[c])) : 1.f;
          x[c] = i > j || (i == j && is_h) ? x[c] * (d * f) : 0.f;
        }
        split_row<NS>(x, [&](int q, int u, const uint4& v) {
          sts128(tile_at<128>(s_t2 + q * Cfg::kMatP, row, t0c / 8 + u), v);
        });
        vec16(kVecBeta, hi);
#pragma unroll
        for (int c = 0; c < 16; ++c) x[c] *= hi[c];
        split_row<NS>(x, [&](int q, int u, const uint4& v) {
          sts128(tile_at<128>(s_t1 + q * Cfg::kMatP, row, t0c / 8 + u), v);
        });
      }
      // the first sums: row of dk, 16 tokens
      tmem_ld(tmem + my, r);
      tmem_ld(tmem + 64 + my, dq);
      tmem_ld(t_w + my, w);
      fence_async();
      umma_fence_before();
      warp_arrive(&mats, lane);
      vec16(kVecEnter, x);
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        dq[c] *= x[c] * p.scale;
        r[c] *= -x[c];
      }
      vec16(kVecLeave, x);
#pragma unroll
      for (int c = 0; c < 16; ++c) w[c] *= x[c];
      wait(&full_kq, k);
      // reads and writes: sums over the 32 of dk, the 32 values over the lanes
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float kv = kq1(t0c + c), qv = kq1(kChunk + t0c + c);
        const float reads = fmaf(qv, dq[c], kv * r[c]), writes = kv * w[c];
        x[c] = (lane & 16 ? writes : reads) + __shfl_xor_sync(0xffffffffu, lane & 16 ? reads : writes, 16);
      }
      over_lanes(x, lane);
      s_rows[buf][quad][lane >> 4][t0c + (lane & 15)] = x[0];
      wait(&done2, k);
      umma_fence_after();
      tmem_ld(t_rq2 + my, x);
#pragma unroll
      for (int c = 0; c < 16; ++c) r[c] += x[c];
      tmem_ld(t_rq2 + 64 + my, x);
#pragma unroll
      for (int c = 0; c < 16; ++c) dq[c] += x[c];
      tmem_ld(t_w2 + my, x);
      const bool parts = p.dq_part != nullptr;
      const int n = row < p.dk ? rows - t0c : 0;  // of the 16 tokens to be written
      const int64_t at = parts ? ((b * p.L + t0 + t0c) * p.heads + h) * p.dk + row
                               : (b * p.L + t0 + t0c) * kstride + (int64_t)hk * p.dk + row;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        w[c] += x[c];
        const float dk = fmaf(beta[t0c + c], w[c], r[c]);
        if (c < n FPSCAN_DEBUG_ONLY(&& grads_within<T, 1>(p, at + c * pstride, at + c * kstride))) {
          if (parts) {
            p.dq_part[at + c * pstride] = dq[c];
            p.dk_part[at + c * pstride] = dk;
          } else {
            static_cast<T*>(p.dq)[at + c * kstride] = Elem<T>::store(dq[c]);
            static_cast<T*>(p.dk_out)[at + c * kstride] = Elem<T>::store(dk);
          }
        }
        x[c] = kq1(t0c + c) * w[c];
      }
      over_lanes(x, lane);
      x[0] += __shfl_xor_sync(0xffffffffu, x[0], 16);
      if (lane < 16) s_rows[buf][quad][2][t0c + lane] = x[0];
      {
        // A's row i (X's or H's share), 16 columns: this thread's [Xb; Hb] times
        // [K; Q] K^T.  Summed over the columns j < t for each t, and that over
        // the rows i >= t.
        const int i = row & 63;
        tmem_ld(t_kk + my, dq);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 a = lds128(tile_at<128>(s_t1, row, t0c / 8 + u));
          const uint4 b = lds128(tile_at<128>(s_t1 + Cfg::kMatP, row, t0c / 8 + u));
          const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            r[8 * u + 2 * e] = bf16_lo(aw[e]) + bf16_lo(bw[e]);
            r[8 * u + 2 * e + 1] = bf16_hi(aw[e]) + bf16_hi(bw[e]);
          }
        }
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          x[c] = i >= t0c + c ? sum : 0.f;
          sum += i > t0c + c ? r[c] * dq[c] : 0.f;
        }
        if (t0c < 48) s_a[buf][t0c / 16][row] = sum;
        over_lanes(x, lane);
        x[0] += __shfl_xor_sync(0xffffffffu, x[0], 16);
        if (lane < 16) s_rows[buf][quad][3][t0c + lane] = x[0];
        umma_fence_before();
      }
      warp_arrive(&used_kq, lane);
    }
  } else if (warp < 19) {
    // ---------------------------------------------------------- <S0, dS>
    // The diagonals of products of 16 x 16 blocks with 8 x 16 ones: most of a
    // product is thrown away, and it still takes a fifth of the instructions
    // of unpacking the parts.
    const int half = warp - 17;
    const int64_t total = mine * strips;
    int64_t next = 0, next_unit = blockIdx.x;  // strip to be copied
    int next_sl = 0;
    Ring<ST> ring, to, left;  // strip at hand, strip to be copied, the strip before the one at hand
    auto load = [&]() {
      const int64_t strip = next_unit * strips + next_sl;
      uint64_t* bar = &full[to.at];
      const uint32_t at = st + Cfg::oRing + to.at * Cfg::kStage;
      __syncwarp();
      if (elect_one()) {
        mbar_expect_tx(bar, Cfg::kTx);
        FPSCAN_DEBUG_ONLY(if (strip_within<NP, NS>(p, strip, strips)) {)
#pragma unroll
        for (int i = 0; i < NP; ++i)
          bulk_in(at + (2 * i + 1) * kStrip, p.do_parts + (strip * NP + i) * (kStrip / 2), kStrip, bar);
#pragma unroll
        for (int i = 0; i < NS; ++i)
          bulk_in(at + i * 2 * kStrip, p.dv_parts + (strip * NS + i) * (kStrip / 2), kStrip, bar);
        bulk_in(at + Cfg::oE, p.e_parts + strip * (NS * kStrip / 2), NS * kStrip, bar);
        bulk_in(at + Cfg::oS, p.s_parts + strip * (NS * kStrip), NS * 2 * kStrip, bar);
        bulk_in(at + Cfg::oD, p.ds_parts + strip * (NS * kStrip), NS * 2 * kStrip, bar);
        FPSCAN_DEBUG_ONLY(})
      }
      __syncwarp();
      ++next;
      to.next();
      if (++next_sl == strips) {
        next_sl = 0;
        next_unit += gridDim.x;
      }
    };
    if (half == 0)
      while (next < min((int64_t)ST, total)) load();
    for (int64_t k = 0; k < mine; ++k) {
      float acc[2][2][4] = {};
      for (int sl = 0; sl < strips; ++sl, ring.next()) {
        const int s = ring.at;
        wait(&full[s], ring.phase);
        const uint32_t at = st + Cfg::oRing + s * Cfg::kStage;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int m0 = (2 * j + half) * 16;
          uint32_t u[2][4], v[2][4];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            ldsm4(u[q], strip_a(at + Cfg::oS + q * 2 * kStrip, lane, m0));
            ldsm4(v[q], strip_b(at + Cfg::oD + q * 2 * kStrip, lane, m0));
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            mma_bf16(acc[j & 1][n], u[1], v[0][2 * n], v[0][2 * n + 1]);
            mma_bf16(acc[j & 1][n], u[0], v[1][2 * n], v[1][2 * n + 1]);
            mma_bf16(acc[j & 1][n], u[0], v[0][2 * n], v[0][2 * n + 1]);
          }
        }
        warp_arrive(&freed[s], lane);
        if (half == 0 && (k > 0 || sl > 0)) {  // the strip before is used up, or nearly
          if (next < total) {
            wait(&freed[left.at], left.phase);
            load();
          }
          left.next();
        }
      }
      const int g = lane >> 2, c = 2 * (lane & 3);
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        dot += (g == c ? acc[j][0][0] + acc[j][1][2] : 0.f) + (g == c + 1 ? acc[j][0][1] + acc[j][1][3] : 0.f);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
      wait(&full_vec[k & 1], k >> 1);  // so the sum of the chunk before the last has been taken
      if (lane == 0) s_dot[k & 1][warp - 17] = dot;
      warp_arrive(&dots[k & 1], lane);
    }
    // no copy may land after the CTA is gone: at once, unless a wait gave up
    if (half == 0)
      for (int64_t j = max((int64_t)0, next - ST); j < next; ++j)
        mbar_wait_soon(&full[j % ST], (uint32_t)((j / ST) & 1));
  } else {
    // ---------------------------------------------------------- K, Q, vectors; a chunk's last sums
    auto load_vec = [&](int64_t k) {
      const int64_t unit = blockIdx.x + k * gridDim.x;
      mbar_expect_tx(&full_vec[k & 1], Cfg::kVecBytes);
      FPSCAN_DEBUG_ONLY(if (vecs_within(p, unit)))
      bulk_in(st + Cfg::oVec + (int)(k & 1) * Cfg::kVecBytes, p.vecs + unit * (kVecCount * kChunk),
              Cfg::kVecBytes, &full_vec[k & 1]);
    };
    auto load_kq = [&](int64_t k) {
      const int64_t unit = blockIdx.x + k * gridDim.x;
      const int64_t bh = unit / p.chunks, chunk = unit - bh * p.chunks, b = bh / p.heads;
      const int hk = (int)(bh - b * p.heads) / (p.heads / p.key_heads);
      const int64_t tile = ((b * p.key_heads + hk) * p.chunks + chunk) * NP * (kTileKQ / 2);
      mbar_expect_tx(&full_kq, NP * kTileKQ);
      FPSCAN_DEBUG_ONLY(if (tile_within<NP>(p, tile)))
      bulk_in(st, p.kq_tiles + tile, NP * kTileKQ, &full_kq);
    };
    __syncwarp();
    if (elect_one()) {
      load_vec(0);
      load_kq(0);
      if (mine > 1) load_vec(1);
    }
    __syncwarp();
    for (int64_t k = 0; k < mine; ++k) {
      const int64_t unit = blockIdx.x + k * gridDim.x;
      const int64_t bh = unit / p.chunks, chunk = unit - bh * p.chunks, b = bh / p.heads;
      const int h = (int)(bh - b * p.heads);
      const int64_t t0 = chunk * kChunk;
      const int rows = (int)min((int64_t)kChunk, p.L - t0);
      const int buf = (int)(k & 1);
      const float* vec = reinterpret_cast<const float*>(dsm + Cfg::oVec + buf * Cfg::kVecBytes);
      bool reset[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 2 * lane + c;
        // a decay of exactly 0 has no slope in its logarithm
        reset[c] = i < rows FPSCAN_DEBUG_ONLY(&& decays_within<T>(p, (b * p.L + t0 + i) * p.heads + h)) &&
                   Elem<T>::load(static_cast<const T*>(p.log_decay)[(b * p.L + t0 + i) * p.heads + h]) < kDecayFloor;
      }
      wait(&full_vec[buf], k >> 1);
      wait(&used_kq, k);
      __syncwarp();
      if (k + 1 < mine && elect_one()) load_kq(k + 1);
      __syncwarp();
      wait(&dots[buf], k >> 1);
      // dbeta, and the sums of dlog_decay: two tokens a lane, in 64 bits
      double reads[2], writes[2], cross[2], state = 0.0;
      float db[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 2 * lane + c;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int o = 0; o < 4; ++o) sum[o] += s_rows[buf][q][o][i];
        reads[c] = sum[0];
        writes[c] = (double)vec[kVecBeta * kChunk + i] * (double)sum[1];
        db[c] = sum[2];
        cross[c] = sum[3];
      }
      // A's columns left of those 16 that t belongs to, rows i >= t
#pragma unroll
      for (int g = 0; g < 3; ++g) {
        double v[2], suffix[2];
        const double none[2] = {0.0, 0.0};
#pragma unroll
        for (int c = 0; c < 2; ++c) v[c] = (double)s_a[buf][g][2 * lane + c] + (double)s_a[buf][g][64 + 2 * lane + c];
        crossing_sums(v, none, lane, suffix);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (g < lane >> 3) cross[c] += suffix[c];
      }
      if (lane < 2) state = (double)vec[kVecEnter * kChunk + kChunk - 1] * (double)s_dot[buf][lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) state += __shfl_xor_sync(0xffffffffu, state, d);
      double out[2];
      crossing_sums(reads, writes, lane, out);
#pragma unroll
      for (int c = 0; c < 2; ++c) out[c] += state + cross[c];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 2 * lane + c;
        if (i < rows) {
          const int64_t o = (b * p.L + t0 + i) * p.heads + h;
          FPSCAN_DEBUG_ONLY(if (!decays_within<T>(p, o)) continue;)
          static_cast<T*>(p.dlog_decay)[o] = Elem<T>::store(reset[c] ? 0.f : (float)out[c]);
          static_cast<T*>(p.dbeta)[o] = Elem<T>::store(db[c]);
        }
      }
      __syncwarp();
      if (k + 2 < mine && elect_one()) load_vec(k + 2);
      __syncwarp();
    }
    mbar_wait_soon(&full_kq, (uint32_t)((mine - 1) & 1));
    for (int64_t k = max((int64_t)0, mine - 2); k < mine; ++k)
      mbar_wait_soon(&full_vec[k & 1], (uint32_t)((k >> 1) & 1));
  }
  umma_fence_before();
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ------------------------------------------------------------------ shared key heads
struct GroupParams {
  const float* src[2];   // (tokens, heads, dk)
  void* dst[2];          // (tokens, key_heads, dk)
  int64_t n;             // tokens x key_heads x dk / 4
  int group, dk4;
};

// Bound by memory: 2 x 2048 tokens, 16 heads in 8 groups, dk = 128: 17 us.
template <typename T>
__global__ void __launch_bounds__(256) delta_group_kernel(const GroupParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int which = blockIdx.x & 1;
  const int64_t step = (int64_t)(gridDim.x / 2) * blockDim.x;
  for (int64_t i = (int64_t)(blockIdx.x / 2) * blockDim.x + threadIdx.x; i < p.n; i += step) {
    const int64_t head = i / p.dk4;
    const int c = (int)(i - head * p.dk4);
    FPSCAN_DEBUG_ONLY(
        if (!within<float>(p.src[which] + (head * p.group * p.dk4 + c) * 4, 4, p.src[which], p.n * p.group * 4) ||
            !within<float>(p.src[which] + ((head + 1) * p.group - 1) * p.dk4 * 4 + c * 4, 4, p.src[which],
                           p.n * p.group * 4) ||
            !within<T, 4 * sizeof(T)>(static_cast<T*>(p.dst[which]) + i * 4, 4, p.dst[which], p.n * 4)) continue;)
    const float4* src = reinterpret_cast<const float4*>(p.src[which]) + head * p.group * p.dk4 + c;
    float4 s = src[0];
    for (int q = 1; q < p.group; ++q) {
      const float4 x = src[(int64_t)q * p.dk4];
      s.x += x.x;
      s.y += x.y;
      s.z += x.z;
      s.w += x.w;
    }
    T* dst = static_cast<T*>(p.dst[which]) + i * 4;
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(dst) = s;
    else
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
  }
}

// ------------------------------------------------------------------ host side
template <typename T, int LV, int C>
cudaError_t launch_rev_as(const DeltaArgs& a, RevParams& r, int64_t bh) {
  using Cfg = RevCfg<T, LV, C>;
  auto kern = delta_rev_kernel<T, LV, C>;
  const cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return e;
  r.slices = (int)((a.dv + 2 * C - 1) / (2 * C));
  return launch_pdl(kern, (unsigned)(bh * r.slices), kRevThreads, Cfg::kSmem, a.stream, r);
}

template <typename T, int LV>
cudaError_t bwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb) {
  constexpr int NP = kParts<T>;
  cudaError_t e = delta_fwd_pass<T, LV>(a, pl, b0, nb, true);
  if (e != cudaSuccess) return e;
  char* ws = static_cast<char*>(a.workspace);
  auto bf = [&](int64_t off) { return reinterpret_cast<__nv_bfloat16*>(ws + off); };
  const int64_t k0 = b0 * a.seqlen * a.key_heads * a.dk, v0 = b0 * a.seqlen * a.heads * a.dv;
  const int64_t g0 = b0 * a.seqlen * a.heads, s0 = b0 * a.heads * a.dv * a.dk;
  const int64_t tok = nb * a.seqlen, bh = nb * a.heads;

  RevParams r{};
  r.kq_tiles = bf(pl.kq_tiles);
  r.grad = static_cast<const T*>(a.grad_out) + v0;
  r.npn = bf(pl.npn);
  r.vecs = reinterpret_cast<const float*>(ws + pl.vecs);
  r.grad_final = a.grad_final ? a.grad_final + s0 : nullptr;
  r.dinitial = a.dinitial ? a.dinitial + s0 : nullptr;
  r.dv_out = static_cast<T*>(a.dv_out) + v0;
  r.do_parts = bf(pl.do_parts);
  r.dv_parts = bf(pl.dv_parts);
  r.ds_parts = bf(pl.ds_parts);
  r.L = a.seqlen;
  r.chunks = pl.chunks;
  r.key_heads = (int)a.key_heads;
  r.heads = (int)a.heads;
  r.dk = (int)a.dk;
  r.dv = (int)a.dv;
  r.scale = a.scale;
  r.nb = nb;
  // as launch_scan chooses
  e = bh * ((a.dv + 31) / 32) <= a.num_sms ? launch_rev_as<T, LV, 16>(a, r, bh)
                                           : launch_rev_as<T, LV, 32>(a, r, bh);
  if (e != cudaSuccess) return e;

  GradParams g{};
  g.kq_tiles = r.kq_tiles;
  g.do_parts = r.do_parts;
  g.e_parts = bf(pl.e_parts);
  g.dv_parts = r.dv_parts;
  g.s_parts = bf(pl.s_parts);
  g.ds_parts = r.ds_parts;
  g.vecs = r.vecs;
  g.log_decay = static_cast<const T*>(a.log_decay) + g0;
  T* dq = static_cast<T*>(a.dq) + k0;
  T* dk = static_cast<T*>(a.dk_out) + k0;
  const bool shared = a.heads != a.key_heads;
  g.dq = dq;
  g.dk_out = dk;
  g.dq_part = shared ? reinterpret_cast<float*>(ws + pl.dq_part) : nullptr;
  g.dk_part = shared ? reinterpret_cast<float*>(ws + pl.dk_part) : nullptr;
  g.dlog_decay = static_cast<T*>(a.dlog_decay) + g0;
  g.dbeta = static_cast<T*>(a.dbeta) + g0;
  g.L = a.seqlen;
  g.chunks = pl.chunks;
  g.units = bh * pl.chunks;
  g.key_heads = (int)a.key_heads;
  g.heads = (int)a.heads;
  g.dk = (int)a.dk;
  g.dv = (int)a.dv;
  g.scale = a.scale;
  g.nb = nb;
  const unsigned grid = (unsigned)std::min<int64_t>(g.units, a.num_sms);
  if constexpr (LV == 1) {
    using GC = TcGradCfg<NP>;
    auto kern = delta_grad_tc_kernel<T>;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GC::kSmem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(kern, grid, kTcThreads, GC::kSmem, a.stream, g);
  } else {
    using GC = GradCfg<NP>;
    auto kern = delta_grad_kernel<T>;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GC::kSmem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(kern, grid, kGradThreads, GC::kSmem, a.stream, g);
  }
  if (e != cudaSuccess || !shared) return e;

  GroupParams s{};
  s.src[0] = g.dq_part;
  s.src[1] = g.dk_part;
  s.dst[0] = dq;
  s.dst[1] = dk;
  s.n = tok * a.key_heads * (a.dk / 4);
  s.group = (int)(a.heads / a.key_heads);
  s.dk4 = (int)(a.dk / 4);
  const unsigned gg = 2 * (unsigned)std::min<int64_t>((s.n + 255) / 256, 8 * a.num_sms);
  return launch_pdl(delta_group_kernel<T>, gg, 256, 0, a.stream, s);
}

template <typename T, int LV>
cudaError_t bwd_all(const DeltaArgs& a, const DeltaPlan& pl) {
  for (int64_t b0 = 0; b0 < a.batch; b0 += pl.batch) {
    const int64_t nb = std::min(pl.batch, a.batch - b0);
    const cudaError_t e = bwd_pass<T, LV>(a, pl, b0, nb);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_delta_bwd(const DeltaArgs& a) {
  const DeltaPlan pl = delta_plan(a.batch, a.seqlen, a.key_heads, a.heads, a.dk, a.dv, a.dtype,
                                  a.wide != 0, true);
  switch (a.dtype) {
    case kF32:
      return bwd_all<float, 2>(a, pl);
    case kF16:
      return a.wide ? bwd_all<__half, 2>(a, pl) : bwd_all<__half, 1>(a, pl);
    default:
      return a.wide ? bwd_all<__nv_bfloat16, 2>(a, pl) : bwd_all<__nv_bfloat16, 1>(a, pl);
  }
}

}  // namespace fpscan
