// Shared device helpers of the gated delta rule kernels (sm_100a).
//
// For one head with a state S of (Dv, Dk) and a = exp(log_decay),
//     e_t = v_t - a_t S_{t-1} k_t,  S_t = a_t S_{t-1} + beta_t e_t k_t^T,
//     o_t = scale S_t q_t.
// The sequence is cut into chunks of C = 64 tokens.  With G the running sum
// of log_decay inside a chunk, D_ij = exp(G_i - G_j), M_ij = D_ij k_i.k_j
// (i > j) and S0 the state entering the chunk:
//     N = (I + M diag(beta))^-1,  E = N (V - exp(G) K S0^T),
//     O = scale exp(G) Q S0^T + P E,   P_ij = scale D_ij (q_i.k_j) beta_j (i >= j),
//     S_C = exp(G_C) S0 + E^T diag(beta exp(G_C - G)) K.
//
// Matrix products run on bf16 tensor-core instructions with fp32 sums.  An
// operand of more than 8 bits is cut into bf16 parts, x = x0 + x1 (+ x2),
// each the rounding of what the parts before it leave, and a product of two
// operands is the sum of the products of their parts i, j with i + j <= LV:
//   LV = 1: relative error near 2^-16 per product, for outputs of 16 bits
//           (a single bf16 rounding, 2^-9, would show in them);
//   LV = 2: near 2^-24, the level of fp32 products, for outputs of 32 bits.
// bf16 inputs are one part, fp16 two, fp32 three, each exactly.  tf32
// products (11 bits) cost as much as LV = 1 and hold less.
#pragma once

#include "common.cuh"

namespace fpscan {

// Debug builds: n elements of type T at p, aligned to ALIGN bytes, inside a
// tensor of `total` elements from `base`.
template <typename T, int ALIGN = 16>
__device__ __forceinline__ bool within(const void* p, int64_t n, const void* base, int64_t total) {
  return in_bounds<ALIGN>(p, n * sizeof(T), base, static_cast<const T*>(base) + total);
}

constexpr int kChunk = 64;
constexpr int kHalfTile = 2 * kChunk * 128;     // bytes: 64 columns of K's, then Q's rows
constexpr int kTileKQ = 2 * kHalfTile;          // one part of K and Q
constexpr int kMatBytes = kChunk * kChunk * 2;  // one part of a 64 x 64 matrix

// Below this log_decay counts as -inf: exp of anything near it is 0, and
// differences of running sums stay finite.
constexpr float kDecayFloor = -10000.f;

// Per-chunk vectors kept by delta_prep_kernel, kChunk floats each.
enum DeltaVec : int {
  kVecEnter = 0,  // exp(G_i)
  kVecLeave = 1,  // exp(G_C - G_i)
  kVecBeta = 2,
  kVecCumHi = 3,  // G_i as a sum of two floats
  kVecCumLo = 4,
  kVecCount = 5
};

template <typename T> constexpr int kParts = 1;
template <> constexpr int kParts<__half> = 2;
template <> constexpr int kParts<float> = 3;

// ---------------------------------------------------------------- tensor-core fragments
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9},"
      " {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// N accumulator tiles of one step (16 values of k) of a product.  The tensor
// core truncates its fp32 sums, and a chain of many truncated sums drifts by
// more than 32-bit results may be off.  So wide products (LV = 2) sum each
// step from zero, smallest parts first, and add it to the accumulator with
// a rounded fp32 add; the others sum in the accumulator itself.
template <bool WIDE, int N>
struct Step {
  float t[WIDE ? N : 1][4];
  __device__ __forceinline__ Step() {
    if constexpr (WIDE) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[n][e] = 0.f;
    }
  }
  __device__ __forceinline__ void mma(int n, float (&acc)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
    if constexpr (WIDE) mma_bf16(t[n], a, b0, b1);
    else mma_bf16(acc, a, b0, b1);
  }
  __device__ __forceinline__ void add(int n, float (&acc)[4]) {
    if constexpr (WIDE) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += t[n][e];
    }
  }
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Tiles in shared memory: rows of ROWB bytes (a multiple of 128), 16-byte
// units exchanged by the low bits of the row, so that 8 rows of one unit
// column (an ldmatrix) fall on 8 different bank groups.
template <int ROWB>
__device__ __forceinline__ uint32_t tile_at(uint32_t base, int row, int unit) {
  return base + row * ROWB + ((unit ^ (row & 7)) << 4);
}

// The four ways a lane addresses an x4 load; `lane` picks the row and unit.
// B operand from [n][k] rows: n tiles n0 and n0 + 8, 16 values of k.
template <int ROWB>
__device__ __forceinline__ uint32_t at_b(uint32_t base, int lane, int n0, int kk) {
  const int m = lane >> 3, r = lane & 7;
  return tile_at<ROWB>(base, n0 + (m >> 1) * 8 + r, kk * 2 + (m & 1));
}
// B operand from [k][n] rows (transposing load): n tiles n0 and n0 + 8.
template <int ROWB>
__device__ __forceinline__ uint32_t at_bt(uint32_t base, int lane, int n0, int kk) {
  const int m = lane >> 3, r = lane & 7;
  return tile_at<ROWB>(base, kk * 16 + (m & 1) * 8 + r, n0 / 8 + (m >> 1));
}
// A operand from [m][k] rows.
template <int ROWB>
__device__ __forceinline__ uint32_t at_a(uint32_t base, int lane, int m0, int kk) {
  const int m = lane >> 3, r = lane & 7;
  return tile_at<ROWB>(base, m0 + (m & 1) * 8 + r, kk * 2 + (m >> 1));
}
// A operand from [k][m] rows (transposing load).
template <int ROWB>
__device__ __forceinline__ uint32_t at_at(uint32_t base, int lane, int m0, int kk) {
  const int m = lane >> 3, r = lane & 7;
  return tile_at<ROWB>(base, kk * 16 + (m >> 1) * 8 + r, m0 / 8 + (m & 1));
}

// Strips: the parts of E, dO, dV (64 tokens) and of S0, dS (128 rows of dk) by
// 16 values, rows of 32 bytes; kept in global memory as they lie in shared
// memory.  Units are exchanged so that 8 rows of one unit column again fall on
// 8 different bank groups: the 32-byte swizzle of tcgen05 operands.
constexpr int kStrip = kChunk * 32;  // bytes of a bf16 strip
__device__ __forceinline__ uint32_t strip_at(uint32_t base, int row, int unit) {
  return base + row * 32 + ((unit ^ ((row >> 2) & 1)) << 4);
}
// A operand with the tokens as its rows (m0..m0+15).
__device__ __forceinline__ uint32_t strip_a(uint32_t base, int lane, int m0) {
  const int m = lane >> 3, r = lane & 7;
  return strip_at(base, m0 + (m & 1) * 8 + r, m >> 1);
}
// B operand with the tokens as its columns n0..n0+15.
__device__ __forceinline__ uint32_t strip_b(uint32_t base, int lane, int n0) {
  const int m = lane >> 3, r = lane & 7;
  return strip_at(base, n0 + (m >> 1) * 8 + r, m & 1);
}
__device__ __forceinline__ void stsm4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// ---------------------------------------------------------------- tcgen05
// Products of the sequential kernels: A and B in shared memory, D (128 rows
// of 2 C values, fp32) in tensor memory, one thread issues.  A tiles have
// rows of 128 bytes, B tiles (rows are k, 2 C values each) rows of 4 C; 16-byte
// units are exchanged by the bits of the row that the descriptors' 128- and
// 64-byte swizzles take (tile_at, val_at); tiles start on 1024-byte
// boundaries.  An A tile serves as K-major operand (rows are the operand's
// rows, 64 values of k in 128 bytes) or, with the transpose bit, as MN-major
// operand (rows are k).
template <int C>
__device__ __forceinline__ uint32_t val_at(uint32_t base, int row, int unit) {
  return C == 32 ? base + row * 128 + ((unit ^ (row & 7)) << 4)
                 : base + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4);
}
// leading: bytes from 64 rows of an MN-major operand to its next 64.
__device__ __forceinline__ uint64_t umma_desc_a(uint32_t addr, uint32_t leading) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)((leading >> 4) & 0x3fff) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// part: bytes from one part of B to the next, which is the next 2 C columns.
template <int C>
__device__ __forceinline__ uint64_t umma_desc_b(uint32_t addr, uint32_t part) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)((part >> 4) & 0x3fff) << 16) |
         ((uint64_t)(8 * 4 * C >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(C == 32 ? 2 : 4) << 61);
}
// fp32 D, bf16 A and B, M = 128, n columns; A, B MN-major where `ta`, `tb`.
__host__ __device__ constexpr uint32_t umma_idesc(bool ta, bool tb, int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((ta ? 1u : 0u) << 15) | ((tb ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// A wait that is short as a rule: tries for a while before it reads the clock
// and the limit (a load from global memory), which take longer than the wait.
__device__ __forceinline__ bool mbar_wait_soon(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 256; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_bounded(bar, parity);
}

// One lane of a whole warp, the same one every time.  The issuing warp takes
// its branch as a warp, so that descriptors stay in uniform registers: issued
// by a lone thread of a divergent branch a product took 100 cycles, twice its
// own time.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                     bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1 : 0)
      : "memory");
}
// The barrier's phase completes when all products issued so far have.
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void umma_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void umma_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// D_j = sum over parts i of A, i < NA, i + j <= LV, smallest first, and over KS
// steps of 16 values of k, of A_i B_j: the parts of B lie side by side as
// columns of one product, which costs less than a product for each pair
// (measured cycles of one of 128 rows: 44 for 32 columns, 50 for 64, 66 for
// 128), and each D_j is summed by itself (tmem_sum adds them up).  The first
// product sets all columns, the others are as wide as i + j <= LV asks.
// a_step / b_step are bytes of one step, a_part of one part; b has B's first
// part.  SPLIT: A's steps from the fifth on lie a_half further (K-major tiles
// of 128 columns).  TA: A is MN-major.
template <int C, int NA, int LV, int KS, bool SPLIT, bool TA>
__device__ __forceinline__ void umma_parts(uint32_t d, uint64_t a, uint64_t b, uint32_t a_part,
                                           uint32_t a_step, uint32_t b_step, uint32_t a_half, int ksteps) {
  constexpr int top = (NA < LV + 1 ? NA : LV + 1) - 1;
#pragma unroll
  for (int i = top; i >= 0; --i)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      if (ks < ksteps) {
        const bool first = i == top && ks == 0;
        const uint32_t ao = i * a_part + (SPLIT ? (ks >> 2) * a_half + (ks & 3) * a_step : ks * a_step);
        umma(d, a + (ao >> 4), b + (ks * b_step >> 4),
             umma_idesc(TA, true, 2 * C * (first ? LV + 1 : LV - i + 1)), !first);
      }
}

// 16 or 32 columns of the warp's 32 lanes.
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Tensor memory of two products of 2 C columns for each of the LV + 1 parts (a
// power of two of columns).
template <int LV, int C>
constexpr int kTmemColumns = (LV + 1) * 4 * C <= 128 ? 128 : (LV + 1) * 4 * C <= 256 ? 256 : 512;

// The sum of what umma_parts left in NS times 2 C columns, smallest first.
template <int NS, int C>
__device__ __forceinline__ void tmem_sum(uint32_t addr, float (&x)[C]) {
  tmem_ld(addr + (NS - 1) * 2 * C, x);
#pragma unroll
  for (int j = NS - 2; j >= 0; --j) {
    float y[C];
    tmem_ld(addr + j * 2 * C, y);
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] += y[i];
  }
}

// ---------------------------------------------------------------- bf16 parts
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// P parts of the pair (x, y), each packed as bf16 x 2.
template <int P>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&out)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p) {
    out[p] = pack_bf16(x, y);
    if (p + 1 < P) {
      x -= bf16_lo(out[p]);
      y -= bf16_hi(out[p]);
    }
  }
}

// A-operand parts of 16 columns held as two accumulator tiles.
template <int P>
__device__ __forceinline__ void split_frag(const float (&lo)[4], const float (&hi)[4],
                                           uint32_t (&a)[P][4]) {
  uint32_t t[P];
  split_pair<P>(lo[0], lo[1], t);
#pragma unroll
  for (int p = 0; p < P; ++p) a[p][0] = t[p];
  split_pair<P>(lo[2], lo[3], t);
#pragma unroll
  for (int p = 0; p < P; ++p) a[p][1] = t[p];
  split_pair<P>(hi[0], hi[1], t);
#pragma unroll
  for (int p = 0; p < P; ++p) a[p][2] = t[p];
  split_pair<P>(hi[2], hi[3], t);
#pragma unroll
  for (int p = 0; p < P; ++p) a[p][3] = t[p];
}

// The parts of C values of a row as 16-byte units 0.., handed to
// put(part, unit, value).
template <int P, int C, typename F>
__device__ __forceinline__ void split_row(const float (&x)[C], F put) {
#pragma unroll
  for (int u = 0; u < C / 8; ++u) {
    uint32_t w[4][P];
#pragma unroll
    for (int c = 0; c < 4; ++c) split_pair<P>(x[u * 8 + 2 * c], x[u * 8 + 2 * c + 1], w[c]);
#pragma unroll
    for (int q = 0; q < P; ++q) put(q, u, make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]));
  }
}

template <typename T, int C>
__device__ __forceinline__ void store_row(T* p, int n, const float (&x)[C]
                                          FPSCAN_DEBUG_ONLY(, const void* base, int64_t total)) {
#pragma unroll
  for (int i = 0; i < C / Elem<T>::kVec; ++i)
    if (i * Elem<T>::kVec < n FPSCAN_DEBUG_ONLY(&& within<T>(p + i * Elem<T>::kVec, Elem<T>::kVec, base, total)))
      *reinterpret_cast<uint4*>(p + i * Elem<T>::kVec) = pack_vec<T>(x + i * Elem<T>::kVec);
}

// ---------------------------------------------------------------- asynchronous copies
// 16 bytes global -> shared; zeros when `in` is false (then src is not read).
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's next row of C values of T, fetched a chunk ahead.  16-bit
// rows wait in shared memory (units of the 128 fetching threads side by
// side), copied asynchronously: loads into registers would be waited for at
// the next loop, which the waits on barriers are.  fp32 rows have no room
// there and are loaded.
template <typename T, int C>
struct NextRow {
  static constexpr int V = Elem<T>::kVec, N = C / V;
  static constexpr int kBytes = sizeof(T) == 2 ? 128 * C * 2 : 0;  // of shared memory
  uint4 raw[sizeof(T) == 2 ? 1 : N];
  uint32_t at;
  __device__ __forceinline__ NextRow(uint32_t room, int thread) : at(room + thread * 16) {}
  // the first `n` values (a multiple of 8, may be <= 0) from p, zeros behind them
  __device__ __forceinline__ void fetch(const T* p, int n, const T* valid FPSCAN_DEBUG_ONLY(, int64_t total)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = i * V < n FPSCAN_DEBUG_ONLY(&& within<T>(p + i * V, V, valid, total));
      if constexpr (sizeof(T) == 2)
        cp16(at + i * 128 * 16, in ? p + i * V : valid, in);
      else
        raw[i] = in ? *reinterpret_cast<const uint4*>(p + i * V) : make_uint4(0, 0, 0, 0);
    }
    if constexpr (sizeof(T) == 2) cp_commit();
  }
  __device__ __forceinline__ void take(float (&x)[C]) {
    if constexpr (sizeof(T) == 2) cp_wait<0>();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      Vec16<T> v;
      if constexpr (sizeof(T) == 2)
        v.raw = lds128(at + i * 128 * 16);
      else
        v.raw = raw[i];
#pragma unroll
      for (int c = 0; c < V; ++c) x[i * V + c] = Elem<T>::load(v.e[c]);
    }
  }
};

// The kept tiles move between global and shared memory as they lie there, by
// bulk copies.  Stores: what the warp wrote is made visible to the copy
// engine, then one lane stores and commits; before the bytes are written
// again the lane waits until at most N later groups are unread.
__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// Non-multicast bulk copy to a shared-memory address, completing on `bar`.
__device__ __forceinline__ void bulk_in(uint32_t dst, const void* src, uint32_t bytes,
                                        uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}
// One arrival for a warp whose lanes are done with (or have written) what
// the barrier guards.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  return pack_bf16(x, y);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(bf16_lo(v), bf16_hi(v));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

}  // namespace fpscan
