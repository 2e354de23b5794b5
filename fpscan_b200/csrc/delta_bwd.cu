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
//     dlog_decay_t = sum_{i >= t} (q_i.dQ_i + k_i.R_i - beta_i dbeta_i) + <S_C, dS>.
// The last two hold because beta and k scale a write alike, and because a
// decay scales what is read after it like q and k do: no quotient of a
// gradient by beta or by a decay appears, so zeros of both are harmless.
//
//   delta_split_kernel  fp16 / fp32 only: cuts dO into bf16 parts.
//   delta_rev_kernel    from the last chunk to the first, dS^T in registers
//                       as delta_scan_kernel keeps S^T; writes dV, dS per chunk.
//   delta_grad_kernel   the rest, every (chunk, head) by itself.
//   delta_group_kernel  sums dQ, dK over the heads that share a key head, in
//                       a fixed order.
#include <algorithm>

#include "delta.cuh"
#include "internal.h"

namespace fpscan {

template <typename T, int LV, int DKP>
cudaError_t delta_fwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb,
                           bool keep);

namespace {

// ------------------------------------------------------------------ parts of dO
struct SplitParams {
  const void* src;
  __nv_bfloat16* dst;  // part p at + p * n
  int64_t n;           // elements (a multiple of 8)
};

template <typename T>
__global__ void __launch_bounds__(256) delta_split_kernel(const SplitParams p) {
  constexpr int NP = kParts<T>, V = Elem<T>::kVec;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t step = (int64_t)gridDim.x * blockDim.x * 8;
  const T* src = static_cast<const T*>(p.src);
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; i < p.n; i += step) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) {
      Vec16<T> v;
      v.raw = *reinterpret_cast<const uint4*>(src + i + j * V);
#pragma unroll
      for (int c = 0; c < V; ++c) x[j * V + c] = Elem<T>::load(v.e[c]);
    }
    uint32_t w[4][NP];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_pair<NP>(x[2 * j], x[2 * j + 1], w[j]);
#pragma unroll
    for (int q = 0; q < NP; ++q)
      *reinterpret_cast<uint4*>(p.dst + q * p.n + i) = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
  }
}

// ------------------------------------------------------------------ along the chunks, backwards
struct RevParams {
  const __nv_bfloat16* q_tiles;
  const __nv_bfloat16* k_tiles;
  const __nv_bfloat16* grad;  // dO parts in token rows, part p at + p * grad_stride
  int64_t grad_stride;
  const __nv_bfloat16* n_mat;
  const __nv_bfloat16* p_mat;
  const float* vecs;
  const float* grad_final;
  float* dinitial;
  void* dv_out;
  __nv_bfloat16* do_parts;    // strips, as e_parts
  __nv_bfloat16* dv_parts;
  __nv_bfloat16* ds_parts;
  int64_t L, chunks;
  int key_heads, heads, dk, dv, slices;
  float scale;
};

// As in delta_scan_kernel 16 rows of dS^T are shared by three warps: two
// chain warps with half of dk each, and a helper that computes what does not
// need dS -- Z = P^T dO and the sum (scale exp(G) dO)^T Q that joins the
// state -- and leaves both in shared memory.  K, N are loaded by the first
// chain warp, Q, P by the first helper.
template <int NP, int LV, int DKP, int NW>
struct RevCfg {
  static constexpr int NS = LV + 1;
  static constexpr int kTileK = kChunk * DKP * 2;
  static constexpr int kMat = kChunk * kChunk * 2;
  static constexpr int oN = NP * kTileK, oVec = oN + NS * kMat;
  static constexpr int kStageK = oVec + 3 * kChunk * 4;
  static constexpr int oP = NP * kTileK, oEnter = oP + NS * kMat;
  static constexpr int kStageQ = oEnter + 256;
  // of a strip: dO once or twice; dS's parts; two halves of K dS^T, later dV;
  // Z, later dV's parts; the sum that joins the state
  static constexpr int kG = NP * kStrip, kXS = NS * 16 * DKP * 2, kHalf = 8 * 512;
  static constexpr int kZ = NS * kStrip > 8 * 512 ? NS * kStrip : 8 * 512, kSum = DKP / 8 * 512;
  static constexpr int kRoom = 227 * 1024 - 1280;
  static constexpr int kBase = kXS + 2 * kHalf + kZ + kSum;
  // two stages of K, N come first, then two of dO, then two of Q, P
  static constexpr int kStK = NW * (kBase + kG) + 2 * kStageK + kStageQ <= kRoom ? 2 : 1;
  static constexpr int kBufG = NW * (kBase + 2 * kG) + kStK * kStageK + kStageQ <= kRoom ? 2 : 1;
  static constexpr int kWarp = kBufG * kG + kBase;
  static constexpr int kStQ = NW * kWarp + kStK * kStageK + 2 * kStageQ <= kRoom ? 2 : 1;
  static constexpr int oQ = kStK * kStageK, oWarp = oQ + kStQ * kStageQ;
  static constexpr int kSmem = oWarp + NW * kWarp + 128;
  static constexpr bool kFits = kSmem + 1152 <= 227 * 1024;
};

template <typename T, int NP, int LV, int DKP, int NW>
__global__ void __launch_bounds__(NW * 96, 1) delta_rev_kernel(const RevParams p) {
  using Cfg = RevCfg<NP, LV, DKP, NW>;
  static_assert(Cfg::kFits);
  constexpr int NS = Cfg::NS, ROWB = DKP * 2, NT = DKP / 8, MROW = kChunk * 2;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t sm0 = smem_addr(dsm);
  __shared__ __align__(8) uint64_t full_k[2], free_k[2], full_q[2], free_q[2];
  __shared__ __align__(8) uint64_t full_z[NW], free_z[NW], full_g[NW], free_g[NW], pair[NW];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int64_t bh = blockIdx.x / p.slices;
  const int slice = (int)(blockIdx.x - bh * p.slices);
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int dv_cta = slice * NW * 16;
  const int nact = min(NW, (p.dv - dv_cta + 15) / 16);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full_k[i], 1);
      mbar_init(&free_k[i], 2 * nact);
      mbar_init(&full_q[i], 1);
      mbar_init(&free_q[i], nact);
    }
    for (int i = 0; i < NW; ++i) {
      mbar_init(&full_z[i], 1);
      mbar_init(&free_z[i], 2);
      mbar_init(&full_g[i], 1);
      mbar_init(&free_g[i], 2);
      mbar_init(&pair[i], 2);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  const int w = warp < 2 * NW ? warp >> 1 : warp - 2 * NW;  // strip
  const int side = warp & 1;                                // chain: half of dk
  const int dv0 = dv_cta + w * 16, nval = p.dv - dv0;
  const int strips = (p.dv + 15) / 16;
  const int64_t unit0 = bh * p.chunks, tile = (b * p.key_heads + hk) * p.chunks;
  const int64_t vstride = (int64_t)p.heads * p.dv;
  const uint32_t own = sm0 + Cfg::oWarp + w * Cfg::kWarp;
  const uint32_t x_s = own + Cfg::kBufG * Cfg::kG, x_h = x_s + Cfg::kXS, x_z = x_h + 2 * Cfg::kHalf,
                 x_g = x_z + Cfg::kZ;
  // step d handles chunk chunks - 1 - d
  int64_t next = 0;  // steps issued by this loading lane
  auto issue_k = [&]() {
    const int64_t c = p.chunks - 1 - next;
    const int s = (int)(next % Cfg::kStK);
    if (next >= Cfg::kStK && !mbar_wait_bounded(&free_k[s], (uint32_t)((next / Cfg::kStK - 1) & 1)))
      return false;
    const uint32_t st = sm0 + s * Cfg::kStageK;
    mbar_expect_tx(&full_k[s], Cfg::oVec + 3 * kChunk * 4);
    bulk_in(st, p.k_tiles + (tile + c) * NP * (kChunk * DKP), NP * Cfg::kTileK, &full_k[s]);
    bulk_in(st + Cfg::oN, p.n_mat + (unit0 + c) * NS * (kChunk * kChunk), NS * Cfg::kMat, &full_k[s]);
    bulk_in(st + Cfg::oVec, p.vecs + (unit0 + c) * (kVecCount * kChunk), 3 * kChunk * 4, &full_k[s]);
    ++next;
    return true;
  };
  auto issue_q = [&]() {
    const int64_t c = p.chunks - 1 - next;
    const int s = (int)(next % Cfg::kStQ);
    if (next >= Cfg::kStQ && !mbar_wait_bounded(&free_q[s], (uint32_t)((next / Cfg::kStQ - 1) & 1)))
      return false;
    const uint32_t st = sm0 + Cfg::oQ + s * Cfg::kStageQ;
    mbar_expect_tx(&full_q[s], Cfg::oEnter + kChunk * 4);
    bulk_in(st, p.q_tiles + (tile + c) * NP * (kChunk * DKP), NP * Cfg::kTileK, &full_q[s]);
    bulk_in(st + Cfg::oP, p.p_mat + (unit0 + c) * NS * (kChunk * kChunk), NS * Cfg::kMat, &full_q[s]);
    bulk_in(st + Cfg::oEnter, p.vecs + (unit0 + c) * (kVecCount * kChunk), kChunk * 4, &full_q[s]);
    ++next;
    return true;
  };

  if (warp < 2 * NW && nval > 0) {
    // ---------------------------------------------------------- chain
    constexpr int HT = NT / 2;  // tiles of this half
    const int d0 = side * (DKP / 2);
    const bool loads = warp == 0 && lane == 0;
    // dV's tiles, as E's in delta_scan_kernel
    auto e_at = [&](int n) {
      const int blk = n >> 1, of = blk == 0 || blk == 3 ? 0 : 1;
      return x_h + (1 - of) * Cfg::kHalf + ((blk >> 1) * 2 + (n & 1)) * 512 + lane * 16;
    };
    if (loads)
      while (next < min((int64_t)Cfg::kStK, p.chunks)) issue_k();
    __syncwarp();
    float S[HT][4];  // dS^T
#pragma unroll
    for (int n = 0; n < HT; ++n) {
#pragma unroll
      for (int c = 0; c < 4; ++c) S[n][c] = 0.f;
      if (p.grad_final != nullptr) {
        const int dk = d0 + n * 8 + 2 * t4;
        const float* src = p.grad_final + (bh * p.dv + dv0 + g4) * p.dk + dk;
        if (dk < p.dk) {
          const float2 v = *reinterpret_cast<const float2*>(src);
          S[n][0] = v.x;
          S[n][1] = v.y;
          if (nval > 8) {
            const float2 y = *reinterpret_cast<const float2*>(src + 8 * p.dk);
            S[n][2] = y.x;
            S[n][3] = y.y;
          }
        }
      }
    }
    bool ok = true;
    for (int64_t d = 0; d < p.chunks; ++d) {
      const int64_t c = p.chunks - 1 - d;
      const int sk = (int)(d % Cfg::kStK);
      const uint32_t st = sm0 + sk * Cfg::kStageK;
      const float* vec = reinterpret_cast<const float*>(dsm + sk * Cfg::kStageK + Cfg::oVec);
      const float* enter = vec + kVecEnter * kChunk;
      const float* leave = vec + kVecLeave * kChunk;
      const float* beta = vec + kVecBeta * kChunk;
      // one stage: the load waits for every chain warp
      if (Cfg::kStK == 1 && d > 0 && loads) ok = issue_k();
      ok = ok && mbar_wait_bounded(&full_k[sk], (uint32_t)((d / Cfg::kStK) & 1));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const float total = enter[kChunk - 1];

      // Y = (K dS^T)^T: 16 values x 64 tokens, this half of dk.  dS's parts
      // are kept.
      float Y[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) Y[n][e] = 0.f;
#pragma unroll
      for (int k2 = 0; k2 < HT / 2; ++k2) {
        const int kk = side * (HT / 2) + k2;
        uint32_t a[NS][4];
        split_frag<NS>(S[2 * k2], S[2 * k2 + 1], a);
#pragma unroll
        for (int q = 0; q < NS; ++q)
          stsm4(half_a<DKP>(x_s + (side * NS + q) * 16 * DKP, lane, k2), a[q]);
#pragma unroll
        for (int n2 = 0; n2 < 4; ++n2) {
          Step<LV == 2, 2> s;
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t kb[4];
            ldsm4(kb, at_b<ROWB>(st + i * Cfg::kTileK, lane, n2 * 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, Y[2 * n2], a[j], kb[0], kb[1]);
              s.mma(1, Y[2 * n2 + 1], a[j], kb[2], kb[3]);
            }
          }
          s.add(0, Y[2 * n2]);
          s.add(1, Y[2 * n2 + 1]);
        }
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) sts_acc(x_h + side * Cfg::kHalf + n * 512 + lane * 16, Y[n]);
      fence_async();
      __syncwarp();
      if (lane == 0) {
        bulk_s2g(p.ds_parts + (((unit0 + c) * strips + dv0 / 16) * 2 + side) * NS * 8 * DKP,
                 x_s + side * NS * 16 * DKP, NS * 16 * DKP);
        bulk_commit();
        mbar_arrive(&pair[w]);
      }
      // the stage of the chunk before is free by now
      if (Cfg::kStK == 2 && loads && d > 0 && next < p.chunks) ok = issue_k();
      ok = ok && mbar_wait_bounded(&pair[w], 0);
      ok = ok && mbar_wait_bounded(&full_z[w], (uint32_t)(d & 1));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;

      // F = Z + beta exp(G_C - G) Y, in place
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int tok = n * 8 + 2 * t4;
        const float2 lv = *reinterpret_cast<const float2*>(leave + tok);
        const float2 bt = *reinterpret_cast<const float2*>(beta + tok);
        float z[4], y[4];
        lds_acc(x_z + n * 512 + lane * 16, z);
        lds_acc(x_h + (1 - side) * Cfg::kHalf + n * 512 + lane * 16, y);
        const float w0 = lv.x * bt.x, w1 = lv.y * bt.y;
        Y[n][0] = fmaf(w0, Y[n][0] + y[0], z[0]);
        Y[n][1] = fmaf(w1, Y[n][1] + y[1], z[1]);
        Y[n][2] = fmaf(w0, Y[n][2] + y[2], z[2]);
        Y[n][3] = fmaf(w1, Y[n][3] + y[3], z[3]);
      }

      // dV = N^T F, this side's blocks of tokens: 0, 3 or 1, 2
      float V[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) V[n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t a[NS][4];
        split_frag<NS>(Y[2 * kk], Y[2 * kk + 1], a);
        auto block = [&](int n2, float (&v0)[4], float (&v1)[4]) {
          Step<LV == 2, 2> s;
#pragma unroll
          for (int i = LV; i >= 0; --i) {
            uint32_t nb[4];
            ldsm4_t(nb, at_bt<MROW>(st + Cfg::oN + i * Cfg::kMat, lane, n2 * 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, v0, a[j], nb[0], nb[1]);
              s.mma(1, v1, a[j], nb[2], nb[3]);
            }
          }
          s.add(0, v0);
          s.add(1, v1);
        };
        if (kk >= side) block(side, V[0], V[1]);
        if (kk >= 3 - side) block(3 - side, V[2], V[3]);
      }
      // dV's tiles go to the other side; its parts, over Z once both sides
      // have read that, are kept
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n2 = i == 0 ? side : 3 - side;
        sts_acc(e_at(2 * n2), V[2 * i]);
        sts_acc(e_at(2 * n2 + 1), V[2 * i + 1]);
      }
      warp_arrive(&pair[w], lane);
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pair[w], 1));
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n2 = i == 0 ? side : 3 - side;
        uint32_t a[NS][4];
        split_frag<NS>(V[2 * i], V[2 * i + 1], a);
#pragma unroll
        for (int q = 0; q < NS; ++q) stsm4_t(strip_at_t(x_z + q * kStrip, lane, n2), a[q]);
      }
      fence_async();
      __syncwarp();
      if (lane == 0) {
        __nv_bfloat16* vp = p.dv_parts + ((unit0 + c) * strips + dv0 / 16) * NS * (kStrip / 2);
#pragma unroll
        for (int q = 0; q < NS; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n2 = i == 0 ? side : 3 - side;  // 16 rows of 32 bytes
            bulk_s2g(vp + q * (kStrip / 2) + n2 * 256, x_z + q * kStrip + n2 * 512, 512);
          }
        bulk_commit();
      }
      {
        const int64_t t0 = c * kChunk;
        const int rows = (int)min((int64_t)kChunk, p.L - t0);
        T* out = static_cast<T*>(p.dv_out) + (b * p.L + t0) * vstride + (int64_t)h * p.dv + dv0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n2 = i == 0 ? side : 3 - side;
          if constexpr (NP == 1) {  // the first bf16 part is the rounded value
            const int r = n2 * 16 + (lane >> 1), un = lane & 1;
            if (r < rows && un * 8 < nval)
              *reinterpret_cast<uint4*>(out + r * vstride + un * 8) = lds128(strip_at(x_z, r, un));
          } else {
#pragma unroll
            for (int n = 0; n < 2; ++n)
              store_t<T>(out + (int64_t)(n2 * 16 + n * 8) * vstride, vstride, V[2 * i + n], lane,
                         rows - n2 * 16 - n * 8, nval);
          }
        }
      }

      // dS <- exp(G_C) dS + (scale exp(G) dO)^T Q - (exp(G) dV)^T K, this half
      uint32_t uv[4][NS][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        float f[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int n = 2 * kk + half;
          const float2 ge = *reinterpret_cast<const float2*>(enter + n * 8 + 2 * t4);
          if ((kk == side) | (kk == 3 - side)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[half][e] = V[(kk >> 1) * 2 + half][e];
          } else {
            lds_acc(e_at(n), f[half]);
          }
          f[half][0] *= -ge.x;
          f[half][1] *= -ge.y;
          f[half][2] *= -ge.x;
          f[half][3] *= -ge.y;
        }
        split_frag<NS>(f[0], f[1], uv[kk]);
      }
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full_g[w], (uint32_t)(d & 1)));
      if (!ok) break;
#pragma unroll
      for (int n4 = 0; n4 < HT / 4; ++n4) {
        float x[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) lds_acc(x_g + (side * HT + n4 * 4 + n) * 512 + lane * 16, x[n]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          Step<LV == 2, 4> s;
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t b0[4], b1[4];
            ldsm4_t(b0, at_bt<ROWB>(st + i * Cfg::kTileK, lane, d0 + n4 * 32, kk));
            ldsm4_t(b1, at_bt<ROWB>(st + i * Cfg::kTileK, lane, d0 + n4 * 32 + 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, x[0], uv[kk][j], b0[0], b0[1]);
              s.mma(1, x[1], uv[kk][j], b0[2], b0[3]);
              s.mma(2, x[2], uv[kk][j], b1[0], b1[1]);
              s.mma(3, x[3], uv[kk][j], b1[2], b1[3]);
            }
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) s.add(n, x[n]);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[n4 * 4 + n][e] = fmaf(total, S[n4 * 4 + n][e], x[n][e]);
      }
      if (lane == 0) bulk_wait_read<0>();  // dS's and dV's parts: Z may come again
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&free_z[w]);
        mbar_arrive(&free_g[w]);
        mbar_arrive(&free_k[sk]);
      }
    }
    if (lane == 0) bulk_wait_all();
    if (!ok && loads)  // no copy may land after the CTA is gone
      for (int64_t j = max((int64_t)0, next - Cfg::kStK); j < next; ++j)
        mbar_wait_bounded(&full_k[j % Cfg::kStK], (uint32_t)((j / Cfg::kStK) & 1));
    if (ok && p.dinitial != nullptr) {
#pragma unroll
      for (int n = 0; n < HT; ++n) {
        const int dk = d0 + n * 8 + 2 * t4;
        float* dst = p.dinitial + (bh * p.dv + dv0 + g4) * p.dk + dk;
        if (dk < p.dk) {
          *reinterpret_cast<float2*>(dst) = make_float2(S[n][0], S[n][1]);
          if (nval > 8) *reinterpret_cast<float2*>(dst + 8 * p.dk) = make_float2(S[n][2], S[n][3]);
        }
      }
    }
  } else if (warp >= 2 * NW && nval > 0) {
    // ---------------------------------------------------------- helper
    const bool loads = w == 0 && lane == 0;
    if (loads)
      while (next < min((int64_t)Cfg::kStQ, p.chunks)) issue_q();
    __syncwarp();
    auto load_g = [&](int64_t d) {
      const int64_t t0 = (p.chunks - 1 - d) * kChunk;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        load_strip<__nv_bfloat16>(
            own + (int)(d % Cfg::kBufG) * Cfg::kG + i * kStrip,
            p.grad + i * p.grad_stride + (b * p.L + t0) * vstride + (int64_t)h * p.dv + dv0,
            vstride * 2, (int)min((int64_t)kChunk, p.L - t0), min(16, nval) / 8, lane);
      cp_commit();
    };
    if (Cfg::kBufG == 2) load_g(0);
    bool ok = true;
    for (int64_t d = 0; d < p.chunks; ++d) {
      const int64_t c = p.chunks - 1 - d;
      const int sq = (int)(d % Cfg::kStQ);
      const uint32_t st = sm0 + Cfg::oQ + sq * Cfg::kStageQ, gst = own + (int)(d % Cfg::kBufG) * Cfg::kG;
      const float* enter = reinterpret_cast<const float*>(dsm + Cfg::oQ + sq * Cfg::kStageQ + Cfg::oEnter);
      if (lane == 0) bulk_wait_read<0>();  // the strip of the step before has been kept
      __syncwarp();
      if (Cfg::kBufG == 1) load_g(d);
      if (Cfg::kBufG == 2 && d + 1 < p.chunks) {
        load_g(d + 1);
        cp_wait<1>();
      } else {
        cp_wait<0>();
      }
      fence_async();
      __syncwarp();
      if (lane == 0) {
        bulk_s2g(p.do_parts + ((unit0 + c) * strips + dv0 / 16) * NP * (kStrip / 2), gst, NP * kStrip);
        bulk_commit();
      }
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full_q[sq], (uint32_t)((d / Cfg::kStQ) & 1)));
      if (!ok) break;
      float Z[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) Z[n][e] = 0.f;
      uint32_t ug[4][NS][4];  // parts of scale exp(G) dO
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t a[NP][4];
#pragma unroll
        for (int i = 0; i < NP; ++i) ldsm4_t(a[i], strip_at_t(gst + i * kStrip, lane, kk));
#pragma unroll
        for (int n2 = 0; n2 <= kk; ++n2) {
          Step<LV == 2, 2> s;
#pragma unroll
          for (int j = LV; j >= 0; --j) {
            uint32_t pb[4];
            ldsm4_t(pb, at_bt<MROW>(st + Cfg::oP + j * Cfg::kMat, lane, n2 * 16, kk));
#pragma unroll
            for (int i = NP - 1; i >= 0; --i) {
              if (i + j > LV) continue;
              s.mma(0, Z[2 * n2], a[i], pb[0], pb[1]);
              s.mma(1, Z[2 * n2 + 1], a[i], pb[2], pb[3]);
            }
          }
          s.add(0, Z[2 * n2]);
          s.add(1, Z[2 * n2 + 1]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 ge = *reinterpret_cast<const float2*>(enter + kk * 16 + (r >> 1) * 8 + 2 * t4);
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            x += bf16_lo(a[i][r]);
            y += bf16_hi(a[i][r]);
          }
          uint32_t parts[NS];
          split_pair<NS>(x * (ge.x * p.scale), y * (ge.y * p.scale), parts);
#pragma unroll
          for (int q = 0; q < NS; ++q) ug[kk][q][r] = parts[q];
        }
      }
      if (d > 0) ok = mbar_wait_bounded(&free_z[w], (uint32_t)((d - 1) & 1));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll
      for (int n = 0; n < 8; ++n) sts_acc(x_z + n * 512 + lane * 16, Z[n]);
      warp_arrive(&full_z[w], lane);
      if (d > 0) ok = mbar_wait_bounded(&free_g[w], (uint32_t)((d - 1) & 1));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll 2
      for (int n4 = 0; n4 < NT / 4; ++n4) {
        float x[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          Step<LV == 2, 4> s;
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t b0[4], b1[4];
            ldsm4_t(b0, at_bt<ROWB>(st + i * Cfg::kTileK, lane, n4 * 32, kk));
            ldsm4_t(b1, at_bt<ROWB>(st + i * Cfg::kTileK, lane, n4 * 32 + 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, x[0], ug[kk][j], b0[0], b0[1]);
              s.mma(1, x[1], ug[kk][j], b0[2], b0[3]);
              s.mma(2, x[2], ug[kk][j], b1[0], b1[1]);
              s.mma(3, x[3], ug[kk][j], b1[2], b1[3]);
            }
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) s.add(n, x[n]);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) sts_acc(x_g + (n4 * 4 + n) * 512 + lane * 16, x[n]);
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full_g[w]);
        mbar_arrive(&free_q[sq]);
      }
      if (loads && next < p.chunks) ok = issue_q();
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
    cp_wait<0>();
    if (lane == 0) bulk_wait_all();
    if (!ok && loads)
      for (int64_t j = max((int64_t)0, next - Cfg::kStQ); j < next; ++j)
        mbar_wait_bounded(&full_q[j % Cfg::kStQ], (uint32_t)((j / Cfg::kStQ) & 1));
  }
  __syncthreads();  // shared memory outlives every copy into it and out of it
}

// ------------------------------------------------------------------ gradients of a chunk
struct GradParams {
  const __nv_bfloat16* q_tiles;
  const __nv_bfloat16* k_tiles;
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
};

constexpr int kGradThreads = 512;

// 16 warps.  The three 64 x dk sums (dQ, R, W) are cut into tiles of 16 MT
// rows x 16 columns, H and X into tiles of 16 x 16; all stay in registers
// while dO, dV, E, S0 and dS pass once through a ring of bulk copies, KS
// strips of 16 values at a time.  One CTA per SM takes chunk after chunk, and
// the ring runs on into the next chunk during the second phase: with a CTA
// per chunk the copies of a chunk and its products took turns.
template <int NP, int LV, int DKP>
struct GradCfg {
  static constexpr int NS = LV + 1;
  static constexpr int MT = DKP / 64;           // m tiles of a warp in the 64 x dk sums
  static constexpr int kColW = DKP / 16;        // warps side by side there
  static constexpr int kTileK = kChunk * DKP * 2;
  static constexpr int kMat = kChunk * kChunk * 2;
  static constexpr int kRows = 16 * DKP * 2;  // 16 rows of a part of S0 or dS
  static constexpr int kOne = (NP + 2 * NS) * kStrip + 2 * NS * kRows;  // one strip's share
  static constexpr int KS = 1;
  // a stage of the ring
  static constexpr int oV = KS * NP * kStrip;
  static constexpr int oE = oV + KS * NS * kStrip;
  static constexpr int oS = oE + KS * NS * kStrip;
  static constexpr int oD = oS + NS * KS * kRows;
  static constexpr int kStage = oD + NS * KS * kRows;
  static_assert(kStage == KS * kOne);
  // K, Q and the decay vectors; the matrices of the second phase (two at a
  // time where four do not fit); the ring
  static constexpr int oQ = NP * kTileK;
  static constexpr int oVec = 2 * NP * kTileK;
  static constexpr int kVecBytes = kVecCount * kChunk * 4;
  static constexpr int oMats = oVec + (kVecBytes + 127) / 128 * 128;
  static constexpr int kSets = LV == 1 ? 2 : 1;  // of two matrices
  static constexpr int oRing = oMats + kSets * 2 * NS * kMat;
  static constexpr int kRoom = 227 * 1024 - 8192 - 128 - oRing;
  static constexpr int kStages = kRoom / kStage < 4 ? kRoom / kStage : 4;
  static constexpr int kSmem = oRing + kStages * kStage + 128;
  static_assert(kStages >= 1 && kSmem + 8192 <= 227 * 1024);
};

template <typename T, int NP, int LV, int DKP>
__global__ void __launch_bounds__(kGradThreads, 1) delta_grad_kernel(const GradParams p) {
  using Cfg = GradCfg<NP, LV, DKP>;
  constexpr int NS = Cfg::NS, NTH = kGradThreads, ROWB = DKP * 2, MROW = kChunk * 2, KS = Cfg::KS;
  constexpr int MT = Cfg::MT, ST = Cfg::kStages, CW = Cfg::kColW;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t st = smem_addr(dsm);
  __shared__ float s_red[3][CW][kChunk];
  __shared__ float s_dot[NTH / 32];
  __shared__ __align__(8) uint64_t full[ST], freed[ST], full_kq;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int row0 = warp / CW * 16 * MT, col0 = warp % CW * 16;  // in the 64 x dk sums
  const int hr = (warp >> 2) * 16, hc = (warp & 3) * 16;        // in H and X
  // The tiles of H and X above the diagonal are not needed: their 6 warps
  // take <S0, dS> instead, and one of them (thread kLoader) issues the copies.
  const bool lower = hc <= hr;
  constexpr int kLoader = 3 * 32;
  const int above = warp < 4 ? warp - 1 : warp < 8 ? warp - 3 : 5;  // 0..5 among those
  const int64_t kstride = (int64_t)p.key_heads * p.dk;
  const int strips = (p.dv + 15) / 16, slices = (strips + KS - 1) / KS;
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

  // the copies: slice by slice, over this CTA's chunks
  const int64_t mine = (p.units - blockIdx.x + gridDim.x - 1) / gridDim.x;  // chunks of this CTA
  const int64_t total = mine * slices;
  int64_t next = 0;      // slices issued
  int64_t next_unit = blockIdx.x;
  int next_slice = 0;
  auto issue = [&]() {
    const int s = (int)(next % ST);
    if (next >= ST && !mbar_wait_bounded(&freed[s], (uint32_t)((next / ST - 1) & 1))) return false;
    const int64_t unit = next_unit;
    const int v0 = next_slice * KS, n = min(KS, strips - v0);
    const uint32_t at = st + Cfg::oRing + s * Cfg::kStage;
    mbar_expect_tx(&full[s], n * Cfg::kOne);
    bulk_in(at, p.do_parts + (unit * strips + v0) * NP * (kStrip / 2), n * NP * kStrip, &full[s]);
    bulk_in(at + Cfg::oV, p.dv_parts + (unit * strips + v0) * NS * (kStrip / 2), n * NS * kStrip, &full[s]);
    bulk_in(at + Cfg::oE, p.e_parts + (unit * strips + v0) * NS * (kStrip / 2), n * NS * kStrip, &full[s]);
    const int64_t sv = (unit * strips + v0) * NS * 16 * DKP;
    bulk_in(at + Cfg::oS, p.s_parts + sv, n * NS * Cfg::kRows, &full[s]);
    bulk_in(at + Cfg::oD, p.ds_parts + sv, n * NS * Cfg::kRows, &full[s]);
    ++next;
    if (++next_slice == slices) {
      next_slice = 0;
      next_unit += gridDim.x;
    }
    return true;
  };
  auto issue_kq = [&](int64_t unit) {
    const int64_t bh = unit / p.chunks, chunk = unit - bh * p.chunks, b = bh / p.heads;
    const int hk = (int)(bh - b * p.heads) / (p.heads / p.key_heads);
    const int64_t tile = ((b * p.key_heads + hk) * p.chunks + chunk) * NP * (kChunk * DKP);
    mbar_expect_tx(&full_kq, 2 * NP * Cfg::kTileK + Cfg::kVecBytes);
    bulk_in(st, p.k_tiles + tile, NP * Cfg::kTileK, &full_kq);
    bulk_in(st + Cfg::oQ, p.q_tiles + tile, NP * Cfg::kTileK, &full_kq);
    bulk_in(st + Cfg::oVec, p.vecs + unit * (kVecCount * kChunk), Cfg::kVecBytes, &full_kq);
  };
  if (tid == kLoader) {
    while (next < min((int64_t)ST, total)) issue();
    issue_kq(blockIdx.x);
  }

  bool ok = true;
  int64_t it = 0;  // slices consumed
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

    for (int sl = 0; sl < slices; ++sl, ++it) {
      const int s_id = (int)(it % ST), n = min(KS, strips - sl * KS);
      const uint32_t at = st + Cfg::oRing + s_id * Cfg::kStage;
      // refill the stage of the slice before: every warp is done with it, or nearly
      if (tid == kLoader && ST > 1 && it > 0 && next < total) issue();
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[s_id], (uint32_t)((it / ST) & 1)));
      if (!ok) break;
      for (int kk = 0; kk < n; ++kk) {
        const uint32_t a_g = at + kk * NP * kStrip, a_v = at + Cfg::oV + kk * NS * kStrip,
                       a_e = at + Cfg::oE + kk * NS * kStrip;
        // this warp's half of dk in the strip's S0 and dS (plus oS, oD)
        const uint32_t s_half = at + (kk * 2 + col0 / (DKP / 2)) * NS * 16 * DKP;
        if (lower) {
          uint32_t ag[NP][4], av[NS][4];
#pragma unroll
          for (int i = 0; i < NP; ++i) ldsm4(ag[i], strip_a(a_g + i * kStrip, lane, hr));
#pragma unroll
          for (int i = 0; i < NS; ++i) ldsm4(av[i], strip_a(a_v + i * kStrip, lane, hr));
          Step<LV == 2, 4> s;
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
            ldsm4_t(sb[j], half_bt<DKP>(s_half + Cfg::oS + j * 16 * DKP, lane, col0 % (DKP / 2)));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            uint32_t ag[NP][4], av[NS][4];
#pragma unroll
            for (int i = 0; i < NP; ++i) ldsm4(ag[i], strip_a(a_g + i * kStrip, lane, row0 + m * 16));
#pragma unroll
            for (int i = 0; i < NS; ++i) ldsm4(av[i], strip_a(a_v + i * kStrip, lane, row0 + m * 16));
            Step<LV == 2, 4> s;
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
            ldsm4_t(db[j], half_bt<DKP>(s_half + Cfg::oD + j * 16 * DKP, lane, col0 % (DKP / 2)));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            uint32_t ae[NS][4];
#pragma unroll
            for (int i = 0; i < NS; ++i) ldsm4(ae[i], strip_a(a_e + i * kStrip, lane, row0 + m * 16));
            Step<LV == 2, 2> s;
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
      // <S0, dS> over this slice (the same place of every part: swizzle does not matter)
      for (int i = above * 32 + lane; !lower && i < n * Cfg::kRows / 16; i += 6 * 32) {
        float x[8] = {}, y[8] = {};
        // 16-byte piece i % DKP of half i / DKP (16 rows of DKP bytes)
        const uint32_t at_i = at + i / DKP * NS * 16 * DKP + i % DKP * 16;
#pragma unroll
        for (int q = NS - 1; q >= 0; --q) {
          const uint4 u = lds128(at_i + Cfg::oS + q * 16 * DKP);
          const uint4 v = lds128(at_i + Cfg::oD + q * 16 * DKP);
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
    ok = ok && mbar_wait_bounded(&full_kq, (uint32_t)(done & 1));
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
    // registers.  As parts in shared memory with each column times beta (set
    // 0, row operands of dQ and R) or without (set 1, column operands of W).
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
      const uint32_t base = st + Cfg::oMats + (Cfg::kSets == 2 ? set : 0) * 2 * NS * Cfg::kMat;
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
    put_mats(0);
    if (Cfg::kSets == 2) put_mats(1);
    // an element pair of K or Q as fp32 (the sum of its parts)
    auto kq_pair = [&](int off, int row, int col) {
      float2 v = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = NP - 1; i >= 0; --i) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(
            dsm + off + i * Cfg::kTileK + tile_at<ROWB>(0, row, col / 8) + (col % 8) * 2);
        v.x += bf16_lo(w);
        v.y += bf16_hi(w);
      }
      return v;
    };
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
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float2 kv = kq_pair(0, i, col0 + n * 8 + 2 * t4);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            aq[m][n][2 * r + c] *= ge * p.scale;
            ar[m][n][2 * r + c] *= -ge;
            aw[m][n][2 * r + c] *= gl;
            sum = fmaf(aw[m][n][2 * r + c], c ? kv.y : kv.x, sum);
          }
        }
        put_row(2, i, sum);
      }
    __syncthreads();

    // dQ += Hb K, R += Xb K: rows i, columns j <= i
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk * 16 > row0 + 16 * MT - 1) break;
      uint32_t kb[NP][4];
#pragma unroll
      for (int j = 0; j < NP; ++j) ldsm4_t(kb[j], at_bt<ROWB>(st + j * Cfg::kTileK, lane, col0, kk));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Step<LV == 2, 4> s;
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
    if (Cfg::kSets == 1) {
      __syncthreads();
      put_mats(1);
      __syncthreads();
    }
    // W += Hs^T Q + Xd^T K: rows j, columns i >= j
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk * 16 + 15 < row0) continue;
      uint32_t kb[NP][4], qb[NP][4];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        ldsm4_t(kb[j], at_bt<ROWB>(st + j * Cfg::kTileK, lane, col0, kk));
        ldsm4_t(qb[j], at_bt<ROWB>(st + Cfg::oQ + j * Cfg::kTileK, lane, col0, kk));
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Step<LV == 2, 4> s;
#pragma unroll
        for (int i = LV; i >= 0; --i) {
          uint32_t fh[4], fx[4];
          const uint32_t base =
              st + Cfg::oMats + (Cfg::kSets == 2 ? 2 * NS * Cfg::kMat : 0) + i * Cfg::kMat;
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
        float reads = 0.f, writes = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int col = col0 + n * 8 + 2 * t4;
          const float2 kv = kq_pair(0, i, col), qv = kq_pair(Cfg::oQ, i, col);
          const float q0 = aq[m][n][2 * r], q1 = aq[m][n][2 * r + 1];
          const float r0 = ar[m][n][2 * r], r1 = ar[m][n][2 * r + 1];
          const float w0 = aw[m][n][2 * r], w1 = aw[m][n][2 * r + 1];
          reads = fmaf(qv.x, q0, fmaf(qv.y, q1, fmaf(kv.x, r0, fmaf(kv.y, r1, reads))));
          writes = fmaf(kv.x, w0, fmaf(kv.y, w1, writes));
          const float k0 = fmaf(be, w0, r0), k1 = fmaf(be, w1, r1);
          if (i < rows && col < p.dk) {
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
        put_row(0, i, reads);
        put_row(1, i, writes);
      }
    __syncthreads();

    // dbeta, and the suffix sums of dlog_decay: one warp, two tokens a lane, in 64 bits
    if (warp == 0) {
      double dg[2], state = 0.0;
      float db[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 2 * lane + c;
        float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < CW; ++w)
#pragma unroll
          for (int q = 0; q < 3; ++q) sum[q] += s_red[q][w][i];
        db[c] = sum[1];
        dg[c] = (double)sum[0] - (double)beta[i] * (double)sum[1];
        state += (double)beta[i] * (double)sum[2];
      }
      if (lane < NTH / 32) state += (double)enter[kChunk - 1] * (double)s_dot[lane];
      double suffix = dg[0] + dg[1];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_down_sync(0xffffffffu, suffix, d);
        if (lane + d < 32) suffix += o;
        state += __shfl_xor_sync(0xffffffffu, state, d);
      }
      const double out[2] = {suffix + state, suffix - dg[0] + state};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 2 * lane + c;
        if (i < rows) {
          const int64_t o = (b * p.L + t0 + i) * p.heads + h;
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
      mbar_wait_bounded(&full[j % ST], (uint32_t)((j / ST) & 1));
    mbar_wait_bounded(&full_kq, 0);
    mbar_wait_bounded(&full_kq, 1);
  }
}

// ------------------------------------------------------------------ shared key heads
struct GroupParams {
  const float* src[2];   // (tokens, heads, dk)
  void* dst[2];          // (tokens, key_heads, dk)
  int64_t n;             // tokens x key_heads x dk / 4
  int group, dk4;
};

template <typename T>
__global__ void __launch_bounds__(256) delta_group_kernel(const GroupParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int which = blockIdx.x & 1;
  const int64_t step = (int64_t)(gridDim.x / 2) * blockDim.x;
  for (int64_t i = (int64_t)(blockIdx.x / 2) * blockDim.x + threadIdx.x; i < p.n; i += step) {
    const int64_t head = i / p.dk4;
    const int c = (int)(i - head * p.dk4);
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
template <typename T, int LV, int DKP, int NW>
cudaError_t rev_nw(const DeltaArgs& a, RevParams& p, int64_t bh) {
  using Cfg = RevCfg<kParts<T>, LV, DKP, NW>;
  auto kern = delta_rev_kernel<T, kParts<T>, LV, DKP, NW>;
  const cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return e;
  p.slices = (int)((a.dv + NW * 16 - 1) / (NW * 16));
  return launch_pdl(kern, (unsigned)(bh * p.slices), NW * 96, Cfg::kSmem, a.stream, p);
}

template <typename T, int LV, int DKP>
cudaError_t bwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb) {
  constexpr int NP = kParts<T>;
  cudaError_t e = delta_fwd_pass<T, LV, DKP>(a, pl, b0, nb, true);
  if (e != cudaSuccess) return e;
  char* ws = static_cast<char*>(a.workspace);
  auto bf = [&](int64_t off) { return reinterpret_cast<__nv_bfloat16*>(ws + off); };
  const int64_t k0 = b0 * a.seqlen * a.key_heads * a.dk, v0 = b0 * a.seqlen * a.heads * a.dv;
  const int64_t g0 = b0 * a.seqlen * a.heads, s0 = b0 * a.heads * a.dv * a.dk;
  const int64_t tok = nb * a.seqlen, bh = nb * a.heads;

  RevParams r{};
  if constexpr (NP > 1) {
    SplitParams sp{static_cast<const T*>(a.grad_out) + v0, bf(pl.grad_rows), tok * a.heads * a.dv};
    const unsigned grid = (unsigned)std::min<int64_t>((sp.n + 2047) / 2048, 16 * a.num_sms);
    e = launch_pdl(delta_split_kernel<T>, grid, 256, 0, a.stream, sp);
    if (e != cudaSuccess) return e;
    r.grad = sp.dst;
    r.grad_stride = sp.n;
  } else {
    r.grad = static_cast<const __nv_bfloat16*>(a.grad_out) + v0;
  }
  r.q_tiles = bf(pl.q_tiles);
  r.k_tiles = bf(pl.k_tiles);
  r.n_mat = bf(pl.n_mat);
  r.p_mat = bf(pl.p_mat);
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
  // chain warps per CTA as in the forward; where four do not fit, two
  const bool two = !RevCfg<NP, LV, DKP, 4>::kFits || bh * ((a.dv + 31) / 32) <= a.num_sms;
  if constexpr (RevCfg<NP, LV, DKP, 4>::kFits)
    e = two ? rev_nw<T, LV, DKP, 2>(a, r, bh) : rev_nw<T, LV, DKP, 4>(a, r, bh);
  else
    e = rev_nw<T, LV, DKP, 2>(a, r, bh);
  if (e != cudaSuccess) return e;

  GradParams g{};
  g.q_tiles = r.q_tiles;
  g.k_tiles = r.k_tiles;
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
  using GC = GradCfg<NP, LV, DKP>;
  auto kern = delta_grad_kernel<T, NP, LV, DKP>;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GC::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kern, (unsigned)std::min<int64_t>(g.units, a.num_sms), kGradThreads, GC::kSmem,
                 a.stream, g);
  if (e != cudaSuccess || !shared) return e;

  GroupParams s{};
  s.src[0] = g.dq_part;
  s.src[1] = g.dk_part;
  s.dst[0] = dq;
  s.dst[1] = dk;
  s.n = tok * a.key_heads * (a.dk / 4);
  s.group = (int)(a.heads / a.key_heads);
  s.dk4 = (int)(a.dk / 4);
  const unsigned grid = 2 * (unsigned)std::min<int64_t>((s.n + 255) / 256, 8 * a.num_sms);
  return launch_pdl(delta_group_kernel<T>, grid, 256, 0, a.stream, s);
}

template <typename T, int LV>
cudaError_t bwd_all(const DeltaArgs& a, const DeltaPlan& pl) {
  for (int64_t b0 = 0; b0 < a.batch; b0 += pl.batch) {
    const int64_t nb = std::min(pl.batch, a.batch - b0);
    const cudaError_t e = pl.dkp == 64 ? bwd_pass<T, LV, 64>(a, pl, b0, nb)
                                       : bwd_pass<T, LV, 128>(a, pl, b0, nb);
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
