// Attention with a decay for each head (sm_100a):
//     S_t = lam S_{t-1} + k_t v_t^T,      o_t = scale S_t^T q_t,     lam = exp(log_decay[h]).
//
// Chunked form. Over a chunk of 64 tokens with the state X before it,
//     o_i = intra sum_{j <= i} lam^(i-j) (q_i . k_j) v_j + inter lam^(i+1) X^T q_i
//     X'  = lam^n X + kv sum_j lam^(n-1-j) k_j v_j^T                 (n tokens in the chunk)
// so all products are 64-wide matrix products and only X walks along the tokens.
//
// The backward pass is the same operator three times:
//     dq = (q, k, v -> do, v, k) forwards, with the transposed states,
//     dk = (v, do, q) and dv = (k, q, do) from the last token to the first,
// with the reverse recurrence holding lam X instead of X (exponents i and n - j
// instead of i + 1 and n - 1 - j): its state starts as the gradient of the final
// state and ends as the gradient of the initial one. One kernel takes up to three
// such roles side by side, which read the same rows while they are in L2.
//
// Few sequences and heads: the tokens are split into segments. k_decay_chunk in
// its state-only form gives each segment's own contribution to the state,
// k_decay_scan turns these into the state before each segment, and the main
// kernel then runs all segments at once. The backward pass takes the states of
// the forward direction from the forward pass, and dk those of dv, transposed.
//
// All products run on tcgen05 in two groups (K': the chunk's keys decayed to its
// end; P: the decayed and masked scores):
//     D = 64:   S [token, token] = Q K^T, O [token, dv] = Q X;
//               then O = lam^(i+1) O + P V, U [dk, dv] = K'^T V
//     D = 128:  S [token, token] = Q K^T, O2 [dv, token] = X^T Q^T;
//               then O1 [dv, token] = V^T P^T, U [dv, dk] = V^T K'
// With D = 64 the first group runs while K' is written; two (D = 128) or three (D =
// 64) blocks per SM fill each other's gaps during the second. With D = 64 the 64 rows
// of every accumulator are read as matrix fragments (16 lanes per warp), X goes back
// as an operand through shared memory, in the place that P takes later, S lies over U,
// and Q X is scaled in place so that P V adds to it: 128 TMEM columns and 72 KB a
// block. With D = 128 the value dimension fills the 128 lanes, X^T stays with its
// rows' threads and goes back through TMEM, over the columns of U, which is done by
// then, but for its last 8 bits, which find room in shared memory only where K' goes:
// their product is the first of the group, and K' is written behind it, its first part
// over the keys; o = lam^(i+1) O2 + O1 at the end. Rows come by cp.async, each thread
// its 16-byte groups (a reversed role simply reads its rows from the end): with D =
// 128 the state fills the 128 registers that two blocks per SM leave a thread, and a
// form with tensor-map loads, which spilled some, took 17 to 25 % longer.
//
// Measured, forward / backward: 8 x 1024 tokens of 12 heads of 64: 40 / 58 us (the
// 138 MB that they have to move take 21 us); 16385 tokens of 16 heads of 128: 160 /
// 351 us (742 MB, 113 us), of which the states before the segments and the scan are
// 57 us each. With a full grid an SM issues in 48 to 51 % of its cycles and the
// tensor pipe works in 34 to 37 %: bound by the latency of a chunk's chain - products,
// their way out of TMEM, the instructions that decay and split operands, products -
// which the two or three blocks of an SM do not cover in full.
//
// Roundings. Products are bf16 tensor-core products with fp32 sums. Whatever is fp32
// and enters one - decayed keys, decayed scores, the state - does so in three bf16
// parts, which hold all of its 24 bits: the state is an fp32 state, and an output is
// rounded once, to bf16. (Scores and state in two parts, 16 bits: forward / backward 37 /
// 55 us and 148 / 306 us, with ten times as many outputs rounded to the wrong
// neighbour, one in 400.) U is formed apart and added to X once per chunk: the tensor
// cores cut off what does not fit their accumulator, which on a state that grows
// over thousands of tokens would add up.
//
// Every wait is bounded (2 s); one that gives up sets an error word of its GPU
// (decay_error_flag), and its block leaves together, with NaN in its rows and its
// state, and frees its TMEM.
#include "common.cuh"
#include "decoder_api.h"
#include "sm100.cuh"

namespace nexar {

namespace {
using namespace sm100;
constexpr int kChunk = 64;
constexpr uint64_t kDecayWaitNs = 2000000000ull;
__device__ unsigned int g_decay_error = 0;  // set once a wait has given up

NEXAR_D void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // zero-filled where there is no token
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
NEXAR_D void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> NEXAR_D void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Four 8 x 8 fragments stored transposed; lane l gives the address of row l % 8 of matrix l / 8.
NEXAR_D void stsm4t(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};"
               :: "r"(addr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
// The same, not transposed.
NEXAR_D void stsm4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};"
               :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// Packed fp32 pairs: x = x * f + u.
NEXAR_D void fma2(float& x0, float& x1, float f, float u0, float u1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %4};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x0), "+f"(x1) : "f"(f), "f"(u0), "f"(u1));
}
// x, y times f.
NEXAR_D void mul2(float& x, float& y, float f) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\t"
      "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(x), "+f"(y) : "f"(f));
}
NEXAR_D uint32_t bf2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
NEXAR_D float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
NEXAR_D float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// An fp32 value as three bf16 parts: the upper 8 bits of its significand, cut off, then those of the rest, then the
// last 8, so the parts hold all of it. top2 gives a pair's part, split2 also leaves the rest in x, y.
NEXAR_D uint32_t top2(float x, float y) { return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632); }
NEXAR_D uint32_t split2(float& x, float& y) {
  const uint32_t p = top2(x, y);
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "sub.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(__uint_as_float(__float_as_uint(x) & 0xffff0000u)), "f"(__uint_as_float(__float_as_uint(y) & 0xffff0000u)));
  return p;
}

// A tile of 64 rows x D bf16 is D / 64 boxes of 64 rows x 128 bytes in the
// 128-byte-swizzled layout of the tcgen05 descriptors: 16-byte group g of row r.
NEXAR_D uint32_t tile_at(int r, int g) { return (uint32_t)((g >> 3) * 8192 + r * 128 + (((g & 7) ^ (r & 7)) << 4)); }
// MN-major operand: boxes of 64 contiguous MN elements x 64 K rows, 8 KB apart.
NEXAR_D uint64_t desc_mn(uint32_t addr) { return umma_desc_sw128_mnmajor(addr); }
// tcgen05.mma and commit by the elected lane of a converged warp (always the same one). With the election inside,
// the operands stay in uniform registers: 32 products of 64 x 64 x 16 take 1120 cycles instead of the 1570 that one
// lane in a branch of its own needs, and the first four 375 instead of 660.
NEXAR_D void warp_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
NEXAR_D void warp_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :: "r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
NEXAR_D void warp_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      :: "r"(smem_u32(bar)) : "memory");
}
NEXAR_D void tmem_st_x8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 lanes x 32 columns as matrix fragments: r[4 n + e] is row lane / 4 + 8 (e / 2), column 8 n + 2 (lane % 4) + e % 2.
NEXAR_D void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
NEXAR_D void tmem_st_frag(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
         "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
NEXAR_D void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait by polling: these waits sit on the chunk's critical path.
NEXAR_D bool wait_phase(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (globaltimer_ns() - t0 > kDecayWaitNs) return false;
  }
}

template <int D, bool STATES> struct Shape {
  static constexpr int kThreads = 256;             // two warps per TMEM lane quarter share its columns
  static constexpr int kBlocks = D == 64 ? 3 : 2;  // resident per SM
  static constexpr int kTile = kChunk * D * 2;     // bytes of one tile of q, k or v
  static constexpr int kTiles = STATES ? 2 : 3;    // (q,) k, v
  static constexpr int kStages = STATES ? 2 : 1;   // chunks of tiles: the main blocks leave no room for a second
  // Three parts of the decayed keys. Main kernel, D = 128: the first part replaces the keys themselves, and the other
  // two lie where the third part of X^T was.
  static constexpr bool kInPlace = !STATES && D == 128;
  static constexpr int kKeys = kStages * kTiles * kTile;
  static constexpr int kScores = kKeys + (kInPlace ? 2 : 3) * kTile;  // three parts of P (D = 64: first of X), 8 KB each
  static constexpr int kOut = D == 64 ? kKeys : kScores;              // then the output
  static constexpr int kMisc = kScores + (STATES ? 0 : 24576);
  static constexpr int kSmem = kMisc + 512;
  // TMEM columns. U at 0 (D = 64: first S; D = 128: first both parts of X^T); D = 64: O at 64;
  // D = 128: O1 (first S) at 128, O2 at 192.
  static constexpr uint32_t kCols = STATES ? D : 2 * D;
};

template <int D, bool STATES>
__global__ void __launch_bounds__(Shape<D, STATES>::kThreads, Shape<D, STATES>::kBlocks)
    k_decay_chunk(const __grid_constant__ DecayArgs a) {
  using S = Shape<D, STATES>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const DecayRole& R = a.role[blockIdx.z];
  const int bh = blockIdx.x, seg = blockIdx.y;
  const int b = bh / a.H, h = bh % a.H;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = a.lengths ? max(0, min(a.lengths[b], a.T)) : a.T;
  const int tokens = STATES ? a.seg_tokens : a.seg_tokens * a.step;
  const int t_begin = seg * tokens;
  const int t_end = min(a.T, t_begin + tokens);   // index i, counted from the first token of the direction
  const int live = max(0, min(len, t_end) - t_begin);   // tokens of this segment that exist
  const int nchunks = (live + kChunk - 1) / kChunk;

  float* pw = reinterpret_cast<float*>(smem + S::kMisc);  // lam^0 .. lam^64, then what the rounding of lam^64 leaves out:
                                                          // over hundreds of chunks that error would add up
  uint64_t* done = reinterpret_cast<uint64_t*>(smem + S::kMisc + 320);
  uint64_t* s_done = done + 1;
  uint64_t* x_done = done + 2;  // D = 128: the products that read X^T
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kMisc + 344);
  const uint32_t base = smem_u32(smem);

  // A thread moves 16-byte group g0 of rows r0, r0 + kRows, ... of every tile. Token index i sits at row i, or at
  // len - 1 - i when the direction is reversed.
  constexpr int kGroups = D / 8, kRows = S::kThreads / kGroups, kPasses = kChunk / kRows;
  const int r0 = tid / kGroups, g0 = tid % kGroups;
  const uint32_t at0 = tile_at(r0, g0);  // + 128 kRows bytes for kRows rows more
  const int dir = R.reverse ? -1 : 1, origin = R.reverse ? len - 1 : 0;
  auto prefetch = [&](int c, int w0 = 0, int w1 = S::kTiles) {  // tiles w0 .. w1 - 1 (of q, k, v; STATES: k, v)
    const int left = live - c * kChunk - r0;
    const long long t = origin + dir * (t_begin + c * kChunk + r0);
    const uint32_t dst = base + (S::kStages == 2 ? (c & 1) * S::kTiles * S::kTile : 0) + at0;
#pragma unroll
    for (int w = 0; w < S::kTiles; ++w) {
      if (w < w0 || w >= w1) continue;
      const int which = STATES ? w + 1 : w;
      const long long st = which == 0 ? R.qt : which == 1 ? R.kt : R.vt;
      const __nv_bfloat16* src = (which == 0 ? R.q + b * R.qb + h * R.qh
                                  : which == 1 ? R.k + b * R.kb + h * R.kh : R.v + b * R.vb + h * R.vh) + t * st + g0 * 8;
#pragma unroll
      for (int u = 0; u < kPasses; ++u) {
        const bool there = kRows * u < left;
        cp_async16(dst + w * S::kTile + u * kRows * 128, there ? src + u * (dir * kRows * st) : R.k, there);
      }
    }
    cp_commit();
  };
  if (nchunks > 0) prefetch(0);

  if (tid == 0) {
    mbar_init(done, 1);
    mbar_init(s_done, 1);
    mbar_init(x_done, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, S::kCols);
    tmem_relinquish();
  }
  if (tid <= kChunk + 1) {
    const double g = (double)a.log_decay[h], p = tid == 0 ? 1.0 : exp(g * min(tid, kChunk));
    pw[tid] = tid <= kChunk ? (float)p : (float)(p - (double)(float)p);
  }

  // ---- state. D = 64: fragments of X, rows dk = xr (+ 8), columns dv = 32 half + 8 n + xc (+ 1). D = 128: row dv of
  // X^T, columns 64 half .. 64 half + 63.
  const int quarter = warp & 3, half = warp >> 2;
  const int xr = quarter * 16 + (lane >> 2), xc = (lane & 3) * 2;
  const int dv = quarter * 32 + lane, dk0 = half * 64;
  constexpr int kX = D == 64 ? 16 : 64;
  float X[kX];
  auto x_at = [&](int n) {  // element of [dk, dv] that X[n] holds
    return D == 64 ? (xr + ((n >> 1) & 1) * 8) * D + half * 32 + (n >> 2) * 8 + xc + (n & 1) : (dk0 + n) * D + dv;
  };
  auto x_at_t = [&](int n) {  // the same element of the transposed state
    return D == 64 ? (half * 32 + (n >> 2) * 8 + xc + (n & 1)) * D + xr + ((n >> 1) & 1) * 8 : dv * D + dk0 + n;
  };
  const float* x0 = nullptr;
  bool x0_t = false;
  if constexpr (!STATES) {
    if (a.nseg > 1) {
      x0 = R.segments + ((size_t)bh * a.nseg + seg * a.step) * D * D;
      x0_t = !R.seg_own;
    } else if (R.init) {
      x0 = R.init + (size_t)bh * D * D;
      x0_t = R.init_transposed;
    }
  }
#pragma unroll
  for (int n = 0; n < kX; ++n) X[n] = 0.f;
  if (x0) {
    if (D == 128 && x0_t) {  // 256 bytes in a row for each thread
#pragma unroll
      for (int n = 0; n < kX; n += 4) {
        const float4 x = *reinterpret_cast<const float4*>(x0 + x_at_t(n));
        X[n] = x.x, X[n + 1] = x.y, X[n + 2] = x.z, X[n + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int n = 0; n < kX; ++n) X[n] = x0[x0_t ? x_at_t(n) : x_at(n)];
    }
  }
  bool have = x0 != nullptr;  // a state that is known to be zero is not multiplied
  const bool want_final = STATES || (R.final_state != nullptr && a.nseg == 1);
  const int shift = R.reverse ? 0 : 1;  // exponents: i + shift and n - shift - j

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t lanes = tbase + ((uint32_t)(quarter * 32) << 16);
  bool ok = true;

  for (int c = 0; c < nchunks; ++c) {
    const int n_tok = min(kChunk, live - c * kChunk);
    const uint32_t stage = S::kStages == 2 ? (c & 1) * S::kTiles * S::kTile : 0;
    const uint32_t tq = base + stage, tk = tq + (STATES ? 0 : S::kTile), tv = tk + S::kTile;
    const bool update = want_final || c + 1 < nchunks;
    if constexpr (!STATES && D == 64) {
      if (have) {  // ---- the state as an operand: three bf16 parts
#pragma unroll
        for (int n = 0; n < kX; n += 8) {  // two groups of 8 columns, 16 rows
          uint32_t hi[4], mid[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = X[n + 2 * e], y = X[n + 2 * e + 1];
            hi[e] = split2(x, y);
            mid[e] = split2(x, y);
            lo[e] = top2(x, y);
          }
          const uint32_t at = base + S::kScores + tile_at(quarter * 16 + (lane & 15), half * 4 + n / 4 + (lane >> 4));
          stsm4(at, hi);
          stsm4(at + 8192, mid);
          stsm4(at + 16384, lo);
        }
      }
    }
    if constexpr (!STATES && D == 128) {
      if (have) {  // ---- the same, X^T: two parts over U, which everyone has read before the last barrier, the third in
                   // the place of the keys' parts (boxes of 128 rows of 128 bytes)
        unsigned char* row = smem + S::kKeys + half * 16384 + dv * 128;
#pragma unroll
        for (int n = 0; n < kX; n += 16) {
          uint32_t hi[8], mid[8], lo[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float x = X[n + 2 * e], y = X[n + 2 * e + 1];
            hi[e] = split2(x, y);
            mid[e] = split2(x, y);
            lo[e] = top2(x, y);
          }
          tmem_st_x8(lanes + half * 32 + n / 2, hi);
          tmem_st_x8(lanes + 64 + half * 32 + n / 2, mid);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4*>(row + (((n / 8 + i) ^ (dv & 7)) << 4)) =
                make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
        }
        tmem_st_wait();
        tc_fence_before();
      }
    }
    cp_wait<0>();
    fence_proxy_async_smem();
    // tiles (D = 64: and the state) are visible; everyone has read U and the output, and all leave together if a wait gave up
    if (!__syncthreads_and(ok)) {
      ok = false;
      break;
    }
    // K steps of 16 in the descriptors: 32 bytes along a K-major row (+ 2; the next box of 64 is + 512), 16 rows of
    // an MN-major box (+ 128), 8 columns of a TMEM operand.
    if constexpr (!STATES) {
      if (__shfl_sync(0xffffffffu, warp, 0) == 4) {
        tc_fence_after();
        const uint64_t kq = umma_desc_sw128_kmajor(tq), kk = umma_desc_sw128_kmajor(tk);
        if (D == 128 && have) {  // the third part of X^T first: s_done also says that it has been read
          const uint64_t kx = umma_desc_sw128_kmajor(base + S::kKeys);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            warp_mma(tbase + D + 64, kx + (k >> 2) * 1024 + (k & 3) * 2, kq + (k >> 2) * 512 + (k & 3) * 2,
                     umma_idesc_bf16_f32(D, 64), k > 0);
        }
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = (k >> 2) * 512 + (k & 3) * 2;
          warp_mma(tbase + (D == 64 ? 0 : D), kq + o, kk + o, umma_idesc_bf16_f32(64, 64), k > 0);
        }
        if (D == 64 && have) {
          const uint64_t mx = desc_mn(base + S::kScores);
#pragma unroll
          for (int p = 2; p >= 0; --p)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              warp_mma(tbase + 64, kq + k * 2, mx + p * 512 + 128 * k, umma_idesc_bf16_f32(64, 64, false, true), p < 2 || k > 0);
        }
        warp_commit(s_done);
        if (D == 128 && have) {
#pragma unroll
          for (int p = 1; p >= 0; --p)
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              warp_mma_ts(tbase + D + 64, tbase + p * 64 + k * 8, kq + (k >> 2) * 512 + (k & 3) * 2,
                          umma_idesc_bf16_f32(D, 64), 1);
        }
        if constexpr (D == 128) warp_commit(x_done);
      }
      __syncwarp();
    }
    if constexpr (S::kStages == 2) {
      if (c + 1 < nchunks) prefetch(c + 1);
    }
    auto decay_keys = [&] {  // ---- keys decayed to the chunk's end, in bf16 parts
#pragma unroll
      for (int u = 0; u < kPasses; ++u) {
        unsigned char* src = smem + (tk - base) + at0 + u * kRows * 128;
        const uint4 raw = *reinterpret_cast<const uint4*>(src);
        const uint32_t kw[4] = {raw.x, raw.y, raw.z, raw.w};
        const float w = R.kv * pw[max(n_tok - shift - r0 - kRows * u, 0)];  // rows behind the last token are zero
        uint32_t p0[4], p1[4], p2[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float x = bf_lo(kw[q]), y = bf_hi(kw[q]);
          mul2(x, y, w);
          p0[q] = split2(x, y);
          p1[q] = split2(x, y);
          p2[q] = top2(x, y);
        }
        unsigned char* dst = smem + S::kKeys + at0 + u * kRows * 128;
        *reinterpret_cast<uint4*>(S::kInPlace ? src : dst) = make_uint4(p0[0], p0[1], p0[2], p0[3]);
        if (!S::kInPlace) dst += S::kTile;
        *reinterpret_cast<uint4*>(dst) = make_uint4(p1[0], p1[1], p1[2], p1[3]);
        *reinterpret_cast<uint4*>(dst + S::kTile) = make_uint4(p2[0], p2[1], p2[2], p2[3]);
      }
    };
    if (!S::kInPlace && update) decay_keys();
    if constexpr (!STATES) {
      // ---- P: 16 query rows and 32 key columns per warp, up to the diagonal
      if (!wait_phase(s_done, c & 1)) {
        ok = false;
        if (lane == 0) atomicExch(&g_decay_error, 1u);
      }
      tc_fence_after();
      if (D == 64 && have) {  // Q X -> inter lam^(i + shift) Q X, in place
        uint32_t o[16];
        tmem_ld_frag(lanes + 64 + half * 32, o);
        const float f0 = R.inter * pw[xr + shift], f1 = R.inter * pw[xr + 8 + shift];  // xr: here a token
        tmem_ld_wait();
#pragma unroll
        for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * (n & 2 ? f1 : f0));
        tmem_st_frag(lanes + 64 + half * 32, o);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)  // above the diagonal, where the state's parts or the output were
        if (half * 2 + m > quarter) {
          unsigned char* at = smem + S::kScores + tile_at(quarter * 16 + (lane & 15), 4 * half + 2 * m + (lane >> 4));
#pragma unroll
          for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(at + p * 8192) = make_uint4(0, 0, 0, 0);
        }
      if (half * 2 <= quarter && quarter * 16 < n_tok) {
        uint32_t sc[16];
        tmem_ld_frag(lanes + (D == 64 ? 0 : D) + half * 32, sc);
        // lam^15-jj of this thread's four key columns inside a block of 16
        const float cf[4] = {pw[15 - xc], pw[14 - xc], pw[7 - xc], pw[6 - xc]};
        tmem_ld_wait();
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int kb = half * 2 + m;
          if (kb > quarter) continue;
          float P[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) P[n][e] = __uint_as_float(sc[m * 8 + n * 4 + e]);
          if (kb < quarter) {
            const float f0 = R.intra * pw[xr - kb * 16 - 15], f1 = R.intra * pw[xr + 8 - kb * 16 - 15];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              P[n][0] *= f0 * cf[2 * n], P[n][1] *= f0 * cf[2 * n + 1];
              P[n][2] *= f1 * cf[2 * n], P[n][3] *= f1 * cf[2 * n + 1];
            }
          } else {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int gap = (lane >> 2) + (e >> 1) * 8 - (n * 8 + xc + (e & 1));
                P[n][e] = gap >= 0 ? P[n][e] * (R.intra * pw[max(gap, 0)]) : 0.f;
              }
          }
          uint32_t hi[4], mid[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // rows + 8 (e % 2), columns + 8 (e / 2)
            float u = P[e >> 1][2 * (e & 1)], v = P[e >> 1][2 * (e & 1) + 1];
            hi[e] = split2(u, v);
            mid[e] = split2(u, v);
            lo[e] = top2(u, v);
          }
          const uint32_t at = base + S::kScores + tile_at(quarter * 16 + (lane & 15), 2 * kb + (lane >> 4));
          stsm4(at, hi);
          stsm4(at + 8192, mid);
          stsm4(at + 16384, lo);
        }
      }
    }
    if (S::kInPlace && update) decay_keys();
    if (!STATES && D == 64) tmem_st_wait();
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (__shfl_sync(0xffffffffu, warp, 0) == 4) {  // small parts first
      tc_fence_after();
      const uint64_t mv = desc_mn(tv);
      if constexpr (!STATES) {
        constexpr uint32_t id1 = umma_idesc_bf16_f32(D, 64, D == 128, D == 64);
        const uint64_t kp = umma_desc_sw128_kmajor(base + S::kScores);
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (D == 64)
              warp_mma(tbase + 64, kp + p * 512 + k * 2, mv + 128 * k, id1, p < 2 || k > 0 || have);
            else
              warp_mma(tbase + D, mv + 128 * k, kp + p * 512 + k * 2, id1, p < 2 || k > 0);
          }
      }
      if (update) {
        // D = 128: U takes the columns of X^T. Only products of one accumulator are sure to run in the order of their
        // issue, so those that read X^T are waited for; they were issued a group earlier and have long finished.
        if constexpr (S::kInPlace) {
          if (!wait_phase(x_done, c & 1)) {
            ok = false;
            if (lane == 0) atomicExch(&g_decay_error, 1u);
          }
          tc_fence_after();
        }
        constexpr uint32_t idu = umma_idesc_bf16_f32(D, D, true, true);
        const uint64_t mk = desc_mn(base + S::kKeys);
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t part = (S::kInPlace ? (p ? mk + (p - 1) * (S::kTile >> 4) : desc_mn(tk)) : mk + p * (S::kTile >> 4)) + 128 * k;
            warp_mma(tbase, D == 64 ? part : mv + 128 * k, D == 64 ? mv + 128 * k : part, idu, p < 2 || k > 0);
          }
      }
      warp_commit(done);
    }
    __syncwarp();
    if constexpr (!STATES && D == 64) {
      if (c + 1 < nchunks) prefetch(c + 1, 0, 2);  // nothing reads q and k any more
    }
    if (!wait_phase(done, c & 1)) {
      ok = false;
      if (lane == 0) atomicExch(&g_decay_error, 1u);
    }
    tc_fence_after();
    if constexpr (S::kStages == 1) {
      if (c + 1 < nchunks && ok) prefetch(c + 1, D == 64 ? 2 : 0, 3);
    }
    if (update) {
      const float keep = pw[n_tok], rest = n_tok == kChunk ? pw[kChunk + 1] : 0.f;
#pragma unroll
      for (int n = 0; n < kX; n += 16) {
        uint32_t u[16];
        if constexpr (D == 64) tmem_ld_frag(lanes + half * 32, u);
        else tmem_ld_32x32b_x16(lanes + dk0 + n, u);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float r0_ = X[n + e], r1_ = X[n + e + 1];
          fma2(r0_, r1_, rest, __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
          fma2(X[n + e], X[n + e + 1], keep, r0_, r1_);
        }
      }
    }
    if constexpr (!STATES) {
      // ---- the output, through the space of the keys or of P so that whole 16-byte groups are stored
      unsigned char* o_tile = smem + S::kOut;
      const long long row = origin + dir * (t_begin + c * kChunk);
      __nv_bfloat16* out = R.out + b * R.ob + h * R.oh;
      if constexpr (D == 64) {
        uint32_t o[16];
        tmem_ld_frag(lanes + 64 + half * 32, o);
        tmem_ld_wait();
#pragma unroll
        for (int n = 0; n < 16; n += 2)
          *reinterpret_cast<uint32_t*>(o_tile + tile_at(xr + (n & 2) * 4, half * 4 + (n >> 2)) + xc * 2) =
              bf2(__uint_as_float(o[n]), __uint_as_float(o[n + 1]));
        __syncwarp();  // a warp stores what it wrote: 16 rows of 64 bytes
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = quarter * 16 + u * 8 + (lane >> 2), g = half * 4 + (lane & 3);
          if (r < n_tok)
            *reinterpret_cast<uint4*>(out + (row + dir * r) * R.ot + g * 8) =
                *reinterpret_cast<const uint4*>(o_tile + tile_at(r, g));
        }
      } else {
        // fragments of 16 value rows x 8 tokens, stored transposed
        float f[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) f[n] = have ? R.inter * pw[half * 32 + (n >> 1) * 8 + xc + (n & 1) + shift] : 0.f;
#pragma unroll
        for (int hl = 0; hl < 2; ++hl) {
          const uint32_t from = lanes + ((uint32_t)(hl * 16) << 16) + D + half * 32;
          uint32_t o1[16], o2[16], w[8];
          tmem_ld_frag(from, o1);
          if (have) tmem_ld_frag(from + 64, o2);
          tmem_ld_wait();
#pragma unroll
          for (int n = 0; n < 16; n += 2) {
            float x = __uint_as_float(o1[n]), y = __uint_as_float(o1[n + 1]);
            if (have) {
              x = fmaf(f[(n >> 2) * 2], __uint_as_float(o2[n]), x);
              y = fmaf(f[(n >> 2) * 2 + 1], __uint_as_float(o2[n + 1]), y);
            }
            w[n >> 1] = bf2(x, y);
          }
#pragma unroll
          for (int n = 0; n < 4; n += 2) {
            const int t = half * 32 + (n + (lane >> 4)) * 8 + (lane & 7), g = quarter * 4 + hl * 2 + ((lane >> 3) & 1);
            stsm4t(smem_u32(o_tile) + tile_at(t, g), w[2 * n], w[2 * n + 1], w[2 * n + 2], w[2 * n + 3]);
          }
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();  // the next chunk's X^T goes over columns of U that other warps have read
#pragma unroll
        for (int u = 0; u < kPasses; ++u) {
          const int r = r0 + kRows * u;
          if (r < n_tok)
            *reinterpret_cast<uint4*>(out + (row + dir * r) * R.ot + g0 * 8) =
                *reinterpret_cast<const uint4*>(o_tile + at0 + u * kRows * 128);
        }
      }
      have = true;
    }
    tc_fence_before();
  }

  ok = __syncthreads_and(ok);
  if constexpr (!STATES) {
    // rows of the batch that hold no token (index >= length) give zeros; where a wait gave up, all are NaN
    __nv_bfloat16* rows = R.out + b * R.ob + h * R.oh;
    const uint32_t fill = ok ? 0u : 0x7fc07fc0u;
    const int from = ok ? max(t_begin, min(len, t_end)) : t_begin;
    for (int e = tid; e < (t_end - from) * kGroups; e += S::kThreads) {
      const int i = from + e / kGroups;
      *reinterpret_cast<uint4*>(rows + (long long)(i < len ? origin + dir * i : i) * R.ot + (e % kGroups) * 8) =
          make_uint4(fill, fill, fill, fill);
    }
  }
  if (want_final) {
    float* dst = STATES ? R.segments + ((size_t)bh * a.nseg + seg) * D * D : R.final_state + (size_t)bh * D * D;
#pragma unroll
    for (int n = 0; n < kX; ++n) dst[x_at(n)] = ok ? X[n] : __int_as_float(0x7fc00000);
  }
  cp_wait<0>();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tbase, S::kCols);
  }
}

// Segments' own contributions -> the state before each segment, in place, and
// the state behind the last. One thread per 4 elements of a head's state.
template <int D> __global__ void __launch_bounds__(256) k_decay_scan(const __grid_constant__ DecayArgs a) {
  const DecayRole& R = a.role[blockIdx.z];
  const int bh = blockIdx.x, b = bh / a.H, h = bh % a.H;
  const int e = blockIdx.y * 256 + threadIdx.x;  // < D * D / 4
  const int len = a.lengths ? max(0, min(a.lengths[b], a.T)) : a.T;
  // whole segments, then one with the last tokens, then empty ones
  __shared__ float decay[3];
  const int whole = len / a.seg_tokens, rest = len - whole * a.seg_tokens;
  if (threadIdx.x < 2) {
    const double f = exp((double)a.log_decay[h] * (threadIdx.x ? rest : a.seg_tokens));
    decay[threadIdx.x] = threadIdx.x && !rest ? 1.f : (float)f;
    if (threadIdx.x == 0) decay[2] = (float)(f - (double)(float)f);
  }
  float4* p = reinterpret_cast<float4*>(R.segments + (size_t)bh * a.nseg * D * D) + e;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (R.init) {
    const float* q = R.init + (size_t)bh * D * D;
    if (R.init_transposed) {
      const int r = e * 4 / D, c = e * 4 % D;
      x = make_float4(q[c * D + r], q[(c + 1) * D + r], q[(c + 2) * D + r], q[(c + 3) * D + r]);
    } else {
      x = reinterpret_cast<const float4*>(q)[e];
    }
  }
  __syncthreads();
  const float full = decay[0], part = decay[1], full_rest = decay[2];
  constexpr int kBatch = 8;  // segments whose loads are in flight together
  for (int s0 = 0; s0 < a.nseg; s0 += kBatch) {
    float4 u[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (s0 + k < a.nseg) u[k] = p[(size_t)(s0 + k) * (D * D / 4)];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int s = s0 + k;
      if (s < a.nseg) {
        const float f = s < whole ? full : (s == whole ? part : 1.f), r = s < whole ? full_rest : 0.f;
        p[(size_t)s * (D * D / 4)] = x;
        x.x = fmaf(f, x.x, fmaf(r, x.x, u[k].x)), x.y = fmaf(f, x.y, fmaf(r, x.y, u[k].y));
        x.z = fmaf(f, x.z, fmaf(r, x.z, u[k].z)), x.w = fmaf(f, x.w, fmaf(r, x.w, u[k].w));
      }
    }
  }
  if (R.final_state) reinterpret_cast<float4*>(R.final_state + (size_t)bh * D * D)[e] = x;
}

// One token: a block per (sequence, head). Each thread holds 4 columns of every
// eighth row (D = 64: 16 threads to a row; D = 128: a warp), updates them in
// place and sums its part of q^T S; bound by reading and writing the state: 192
// sequences of 32 heads of 128 in 119 us, 6.8 TB/s (812 MB). A few heads take 2.2
// us, the latency of one load, one barrier and one store.
template <int D> __global__ void __launch_bounds__(D * 2) k_decay_step(const DecayStepArgs a) {
  constexpr int kRow = D / 4;             // threads per row
  constexpr int kRows = 8;                // rows at a time
  __shared__ float4 red[kRows][kRow];
  __shared__ float sq[D], sk[D];
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const int tid = threadIdx.x, c = tid % kRow, r0 = tid / kRow;
  float4* S = reinterpret_cast<float4*>(a.state + (size_t)blockIdx.x * D * D) + c;
  float4 st[D / kRows];
#pragma unroll
  for (int i = 0; i < D / kRows; ++i) st[i] = __ldcs(S + (size_t)(r0 + i * kRows) * kRow);
  if (tid < D) {
    sq[tid] = __bfloat162float(a.q[b * a.qb + h * a.qh + tid]);
  } else {
    sk[tid - D] = __bfloat162float(a.k[b * a.kb + h * a.kh + tid - D]);
  }
  const __nv_bfloat16* vp = a.v + b * a.vb + h * a.vh + c * 4;
  const float v0 = __bfloat162float(vp[0]), v1 = __bfloat162float(vp[1]), v2 = __bfloat162float(vp[2]),
              v3 = __bfloat162float(vp[3]);
  const float lam = (float)exp((double)a.log_decay[h]);
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < D / kRows; ++i) {
    const int r = r0 + i * kRows;
    const float k = sk[r], q = sq[r];
    float4 x = st[i];
    x.x = lam * x.x + k * v0, x.y = lam * x.y + k * v1, x.z = lam * x.z + k * v2, x.w = lam * x.w + k * v3;
    __stcs(S + (size_t)r * kRow, x);
    o.x += q * x.x, o.y += q * x.y, o.z += q * x.z, o.w += q * x.w;
  }
  red[r0][c] = o;
  __syncthreads();
  if (r0 == 0) {
#pragma unroll
    for (int i = 1; i < kRows; ++i) {
      const float4 t = red[i][c];
      o.x += t.x, o.y += t.y, o.z += t.z, o.w += t.w;
    }
    uint2 p;
    p.x = bf2(a.scale * o.x, a.scale * o.y);
    p.y = bf2(a.scale * o.z, a.scale * o.w);
    *reinterpret_cast<uint2*>(a.o + (size_t)blockIdx.x * D + c * 4) = p;
  }
}

template <int D, bool STATES>
cudaError_t launch_chunks(const DecayArgs& a, int roles, cudaStream_t s) {
  using S = Shape<D, STATES>;
  const cudaError_t e =
      cudaFuncSetAttribute(k_decay_chunk<D, STATES>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  k_decay_chunk<D, STATES><<<dim3(a.B * a.H, STATES ? a.nseg : (a.nseg + a.step - 1) / a.step, roles), S::kThreads, S::kSmem, s>>>(a);
  return cudaGetLastError();
}

template <int D> cudaError_t decay_typed(const DecayArgs& a, cudaStream_t s, int* launches) {
  *launches = 0;
  if (a.nseg > 1) {
    int own = 0;
    while (own < a.nroles && a.role[own].seg_own) ++own;
    if (own > 0) {
      const cudaError_t e = launch_chunks<D, true>(a, own, s);
      if (e != cudaSuccess) return e;
      k_decay_scan<D><<<dim3(a.B * a.H, D * D / 1024, own), 256, 0, s>>>(a);
      *launches += 2;
    }
  }
  *launches += 1;
  return launch_chunks<D, false>(a, a.nroles, s);
}
}  // namespace

unsigned int decay_error_flag() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_decay_error, sizeof(v));
  return v;
}

namespace {
// us of one pass of the main kernel, by what it measured for 37 to 888 blocks of 4
// to 32 chunks (within 8 %, but for 13 % at 148 blocks of 32 chunks of heads of 64): a
// chunk takes 2.35, 3.5 or 4.7 us with one, two or three blocks of heads of 64 on an SM
// and 4.5 or 6.5 us with one or two of heads of 128, to which each wave of blocks and
// the launch add 2 to 2.5 us. The state-only kernel takes half of each.
double pass_us(long long blocks, long long chunks, int D) {
  static const double kChunkUs[2][4] = {{0, 2.35, 3.5, 4.7}, {0, 4.5, 6.5, 6.5}};
  const int slots = 148 * (D == 64 ? 3 : 2);
  const double* us = kChunkUs[D != 64];
  const long long waves = blocks / slots, rest = blocks % slots;
  const double wave = D == 64 ? 2.5 : 2.0;
  return 2.5 + waves * (wave + chunks * us[slots / 148]) + (rest ? wave + chunks * us[(rest + 147) / 148] : 0.);
}
double move_us(long long states, int D) { return states * (double)(D * D * 4) / 5e6; }  // out of L2 for the most part
// States of n segments: written, then read and written by the scan, which has 8 of them in flight.
double states_us(long long heads, long long n, long long chunks, int D) {
  return 0.5 * pass_us(heads * n, chunks, D) + 3 * move_us(heads * n, D) + 5.0 + 0.7 * ((n + 7) / 8);
}
}  // namespace

// Splitting the tokens pays where the heads alone leave SMs idle. Measured whole /
// split, us, heads of 64: 12 of T = 4096: 151 / 28; 60 of T = 1000: 40 / 32; 96 of
// T = 1024: 40 / 42; of 128: 16 of T = 16385: 1143 / 157; 48 of T = 4096: 286 / 119;
// 128 of T = 1024: 74 / 95. With lengths, segments without a token end at once and
// finer ones share the work out better: as many as fill every resident block (60
// heads of 64 with 1 to 1000 tokens: 40 / 27.5).
int decay_segment_chunks(int B, int T, int H, int D, bool ragged) {
  const long long heads = (long long)B * H, chunks = (T + kChunk - 1) / kChunk;
  long long best = chunks;
  double us = pass_us(heads, chunks, D);
  for (const int blocks : {37, 74, 148, 296, 444, 592, 740, 888}) {
    const long long want = blocks / heads < chunks ? blocks / heads : chunks;
    if (want < 2 || (ragged && blocks != 148 * (D == 64 ? 3 : 2))) continue;
    const long long per = (chunks + want - 1) / want, n = (chunks + per - 1) / per;
    const double split = pass_us(heads * n, per, D) + move_us(heads * n, D) + states_us(heads, n, per, D);
    if (n > 1 && split < us) us = split, best = per;
  }
  return (int)best;
}

// The three uses of the backward pass need fewer segments to fill the GPU: a block
// then takes several, the most where that is as fast. Measured whole / split, us,
// heads of 64: 12 of T = 4096: 152 / 46; 48 of T = 4096: 162 / 129; of 128: 16 of
// T = 16385: 1148 / 349; 40 of T = 4096: 285 / 224.
int decay_backward_step(int B, int T, int H, int D, int chunks) {
  const long long heads = (long long)B * H, all = (T + kChunk - 1) / kChunk, n = (all + chunks - 1) / chunks;
  if (n < 2) return 0;
  double us = pass_us(heads * 3, all, D) - states_us(heads, n, chunks, D);
  int best = 0;
  for (int step = n < 16 ? (int)n - 1 : 16; step >= 1; --step) {
    const long long blocks = heads * 3 * ((n + step - 1) / step);
    const double split = pass_us(blocks, (long long)step * chunks, D) + move_us(blocks, D);
    if (split < us) us = split, best = step;
  }
  return best;
}

cudaError_t decay_attention(const DecayArgs& a, cudaStream_t s, int* launches) {
  if (a.nroles < 1 || a.nroles > 3 || a.B < 1 || a.H < 1 || a.T < 1 || (long long)a.B * a.H > 0x7fffffffLL || a.nseg > 65535 || a.nseg < 1 || a.step < 1 ||
      (long long)a.nseg * a.seg_tokens < a.T || (a.nseg > 1 && a.seg_tokens % kChunk))
    return cudaErrorInvalidValue;
  if (a.D == 64) return decay_typed<64>(a, s, launches);
  if (a.D == 128) return decay_typed<128>(a, s, launches);
  return cudaErrorInvalidValue;
}

cudaError_t decay_step(const DecayStepArgs& a, cudaStream_t s) {
  const long long blocks = (long long)a.B * a.H;
  if (blocks < 1 || blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (a.D == 64)
    k_decay_step<64><<<(unsigned)blocks, 128, 0, s>>>(a);
  else if (a.D == 128)
    k_decay_step<128><<<(unsigned)blocks, 256, 0, s>>>(a);
  else
    return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace nexar
