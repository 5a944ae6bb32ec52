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
// kernel then runs all segments at once.
//
// Rows come by TMA in their order; a reversed role numbers them from the end.
// All products run on tcgen05 in two groups (K': the chunk's keys decayed to its
// end; P: the decayed and masked scores):
//     D = 64:   S [token, token] = Q K^T, O [token, dv] = Q X;
//               then O = lam^(i+1) O + P V, U [dk, dv] = K'^T V
//     D = 128:  S [token, token] = Q K^T;
//               then O2 [dv, token] = X^T Q^T, O1 [dv, token] = V^T P^T, U [dv, dk] = V^T K'
// The first group runs while K' is written; two (D = 128) or three (D = 64) blocks
// per SM fill each other's gaps during the second. The warp that has no scores above
// the mask issues the products and the loads. With D = 64 the 64 rows of every
// accumulator are read as matrix fragments (16 lanes per warp), X goes back as an
// operand through shared memory, in the place that P takes later, S lies over U, and
// Q X is scaled in place so that P V adds to it: 128 TMEM columns and 64 KB a block.
// With D = 128 the value dimension fills the 128 lanes, X^T stays with its rows'
// threads and goes back through TMEM, over the columns of U, which is done by then;
// o = lam^(i+1) O2 + O1 at the end.
//
// Roundings. Products are bf16 tensor-core products with fp32 sums. The decayed
// keys that enter the state are split into three bf16 parts (24 bits, all of an
// fp32 value), so the state is an fp32 state; scores and states that enter the
// bf16 output are split into two parts (16 bits), well below the output's
// rounding. U is formed apart and added to X once per chunk: the tensor cores cut
// off what does not fit their accumulator, which on a state that grows over
// thousands of tokens would add up.
//
// Every wait is bounded (2 s); one that gives up sets an error word of its GPU
// (decay_error_flag), the block leaves together and frees its TMEM.
#include "common.cuh"
#include "decoder_api.h"
#include "gemm_api.h"
#include "sm100.cuh"

namespace nexar {

namespace {
using namespace sm100;
constexpr int kChunk = 64;
constexpr uint64_t kDecayWaitNs = 2000000000ull;
__device__ unsigned int g_decay_error = 0;  // set once a wait has given up

// Box of 64 tokens x 64 columns (x = 0 or 64) of head h and sequence b.
NEXAR_D void tma_load_rows(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int h, int t, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(h), "r"(t), "r"(b)
      : "memory");
}
// Four 8 x 8 fragments stored transposed; lane l gives the address of row l % 8 of matrix l / 8.
NEXAR_D void stsm4t(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};"
               :: "r"(addr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
// Packed fp32 pairs: x = x * f + u.
NEXAR_D void fma2(float& x0, float& x1, float f, float u0, float u1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %4};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x0), "+f"(x1) : "f"(f), "f"(u0), "f"(u1));
}
NEXAR_D uint32_t bf2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
NEXAR_D float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
NEXAR_D float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// A tile of 64 rows x D bf16 is D / 64 boxes of 64 rows x 128 bytes in the
// 128-byte-swizzled layout of the tcgen05 descriptors: 16-byte group g of row r.
NEXAR_D uint32_t tile_at(int r, int g) { return (uint32_t)((g >> 3) * 8192 + r * 128 + (((g & 7) ^ (r & 7)) << 4)); }
// MN-major operand: boxes of 64 contiguous MN elements x 64 K rows, 8 KB apart.
NEXAR_D uint64_t desc_mn(uint32_t addr) { return umma_desc_sw128_mnmajor(addr); }
// kind::f16 MMA whose A operand is read from tensor memory.
NEXAR_D void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :: "r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
NEXAR_D void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
         "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
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

// Bounded wait of a whole warp: one lane polls, then every lane sees the completed
// phase itself (a phase that is usually complete costs one test).
NEXAR_D bool wait_phase(uint64_t* bar, uint32_t parity, int lane) {
  if (mbar_try_wait(bar, parity)) return true;
  int ok = 1;
  if (lane == 0) {
    const unsigned long long t0 = globaltimer_ns();
    bool got = false;
    while (!got && ok) {
#pragma unroll 1
      for (int i = 0; i < 64 && !got; ++i) got = mbar_try_wait(bar, parity);
      if (!got && globaltimer_ns() - t0 > kDecayWaitNs) ok = 0;
    }
  }
  ok = __shfl_sync(0xffffffffu, ok, 0);
  if (ok) mbar_try_wait(bar, parity);
  return ok != 0;
}

struct DecayMaps {
  CUtensorMap in[4];
};

template <int D, bool STATES> struct Shape {
  static constexpr int kThreads = 256;             // two warps per TMEM lane quarter share its columns
  static constexpr int kBlocks = D == 64 ? 3 : 2;  // resident per SM
  static constexpr int kTile = kChunk * D * 2;     // bytes of one tile of q, k or v
  static constexpr int kTiles = STATES ? 2 : 3;    // (q,) k, v
  static constexpr int kStages = STATES ? 2 : 1;   // chunks of tiles: the main blocks leave no room for a second
  static constexpr int kKeys = kStages * kTiles * kTile;  // three parts of the decayed keys; then the output
  static constexpr int kScores = kKeys + 3 * kTile;       // two parts of P (D = 64: first of X), 8 KB each
  static constexpr int kMisc = kScores + (STATES ? 0 : 16384);
  static constexpr int kSmem = kMisc + 512;
  // TMEM columns. U at 0 (D = 64: first S; D = 128: first both parts of X^T); D = 64: O at 64;
  // D = 128: O1 (first S) at 128, O2 at 192.
  static constexpr uint32_t kCols = STATES ? D : 2 * D;
};

template <int D, bool STATES>
__global__ void __launch_bounds__(Shape<D, STATES>::kThreads, Shape<D, STATES>::kBlocks)
    k_decay_chunk(const __grid_constant__ DecayArgs a, const __grid_constant__ DecayMaps maps) {
  using S = Shape<D, STATES>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const DecayRole& R = a.role[blockIdx.z];
  const int bh = blockIdx.x, seg = blockIdx.y;
  const int b = bh / a.H, h = bh % a.H;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = a.lengths ? max(0, min(a.lengths[b], a.T)) : a.T;
  const int t_begin = seg * a.seg_tokens;
  const int t_end = min(a.T, t_begin + a.seg_tokens);   // index i, counted from the first token of the direction
  const int live = max(0, min(len, t_end) - t_begin);   // tokens of this segment that exist
  const int nchunks = (live + kChunk - 1) / kChunk;
  const bool rev = R.reverse != 0;

  float* pw = reinterpret_cast<float*>(smem + S::kMisc);  // lam^0 .. lam^64, then what the rounding of lam^64 leaves out:
                                                          // over hundreds of chunks that error would add up
  uint64_t* done = reinterpret_cast<uint64_t*>(smem + S::kMisc + 320);  // second group of products
  uint64_t* s_done = done + 1;                                          // first group
  uint64_t* full = done + 2;                                            // [stage] tiles
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kMisc + 352);
  const uint32_t base = smem_u32(smem);

  // Row r of chunk c's tiles is token first_row(c) + r: index 64 c + r of the segment, or (reversed) 64 c + 63 - r.
  const auto first_row = [&](int c) { return rev ? len - t_begin - (c + 1) * kChunk : t_begin + c * kChunk; };
  // The loads of chunk c's tiles from w0 to w1 (of q, k, v; STATES: k, v), by one thread; rows outside the tensor are
  // filled with zeros. The first call of a chunk announces all its bytes.
  const auto load = [&](int c, int w0, int w1) {
    const int s = S::kStages == 2 ? c & 1 : 0, t0 = first_row(c);
    const uint32_t dst = base + s * S::kTiles * S::kTile;
    if (w0 == 0) mbar_arrive_expect_tx(full + s, S::kTiles * S::kTile);
    for (int w = w0; w < w1; ++w) {
      const int which = STATES ? w + 1 : w;
      const CUtensorMap* m = &maps.in[which == 0 ? R.q : which == 1 ? R.k : R.v];
#pragma unroll
      for (int x = 0; x < D; x += 64) tma_load_rows(dst + w * S::kTile + (x >> 6) * 8192, m, full + s, x, h, t0, b);
    }
  };
  if (tid == 0) {
    mbar_init(done, 1);
    mbar_init(s_done, 1);
    mbar_init(full, 1);
    mbar_init(full + 1, 1);
    mbar_fence_init();
    if (nchunks > 0) load(0, 0, S::kTiles);
    if (S::kStages == 2 && nchunks > 1) load(1, 0, S::kTiles);
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
      const bool own = R.segments_from < 0;
      x0 = (own ? R.segments : a.role[R.segments_from].segments) + ((size_t)bh * a.nseg + seg) * D * D;
      x0_t = !own;
    } else if (R.init) {
      x0 = R.init + (size_t)bh * D * D;
      x0_t = R.init_transposed;
    }
  }
#pragma unroll
  for (int n = 0; n < kX; ++n) X[n] = !x0 ? 0.f : x0[x0_t ? x_at_t(n) : x_at(n)];
  bool have = x0 != nullptr;  // a state that is known to be zero is not multiplied
  const bool want_final = STATES || (R.final_state != nullptr && a.nseg == 1);
  const int shift = rev ? 0 : 1;  // exponents: i + shift and n - shift - j

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  const uint32_t lanes = tbase + ((uint32_t)(quarter * 32) << 16);
  constexpr int kGroups = D / 8, kRows = S::kThreads / kGroups, kPasses = kChunk / kRows;
  const int r0 = tid / kGroups, g0 = tid % kGroups;  // 16-byte group g0 of rows r0, r0 + kRows, ... of a tile
  const uint32_t at0 = tile_at(r0, g0);              // + 128 kRows bytes for kRows rows more
  bool ok = true;
  int seen = 0;  // chunks whose loads were waited for
  const bool ctl = warp == (rev ? 3 : 4) && lane == 0;  // issues products and loads: no scores of this warp are kept
  const auto give_up = [&]() {
    ok = false;
    if (lane == 0) atomicExch(&g_decay_error, 1u);
  };

  for (int c = 0; c < nchunks; ++c) {
    const int n_tok = min(kChunk, live - c * kChunk);
    const int lo = rev ? kChunk - n_tok : 0, hi = rev ? kChunk : n_tok;  // rows [lo, hi) are tokens of this chunk
    const uint32_t stage = S::kStages == 2 ? (c & 1) * S::kTiles * S::kTile : 0;
    const uint32_t tq = base + stage, tk = tq + (STATES ? 0 : S::kTile), tv = tk + S::kTile;
    const bool update = want_final || c + 1 < nchunks;
    if constexpr (!STATES && D == 64) {
      if (have) {  // ---- the state as an operand: two bf16 parts
#pragma unroll
        for (int n = 0; n < kX; n += 2) {
          const uint32_t hi_ = bf2(X[n], X[n + 1]), lo_ = bf2(X[n] - bf_lo(hi_), X[n + 1] - bf_hi(hi_));
          unsigned char* at = smem + S::kScores + tile_at(xr + (n & 2) * 4, half * 4 + (n >> 2)) + xc * 2;
          *reinterpret_cast<uint32_t*>(at) = hi_;
          *reinterpret_cast<uint32_t*>(at + 8192) = lo_;
        }
        fence_proxy_async_smem();
      }
    }
    // The state is written (D = 64); everyone has read U and the output. All leave together if a wait gave up.
    if (!__syncthreads_and(ok)) {
      ok = false;
      break;
    }
    if (!wait_phase(full + (S::kStages == 2 ? c & 1 : 0), (S::kStages == 2 ? c >> 1 : c) & 1, lane)) give_up();
    else seen = c + 1;
    // K steps of 16 in the descriptors: 32 bytes along a K-major row (+ 2; the next box of 64 is + 512), 16 rows of
    // an MN-major box (+ 128), 8 columns of a TMEM operand. Small parts first.
    if constexpr (!STATES) {
      if (ctl) {
        tc_fence_after();
        const uint64_t kq = umma_desc_sw128_kmajor(tq), kk = umma_desc_sw128_kmajor(tk);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = (k >> 2) * 512 + (k & 3) * 2;
          umma_f16(tbase + (D == 64 ? 0 : 128), kq + o, kk + o, umma_idesc_bf16_f32(64, 64), k > 0);
        }
        if (D == 64 && have) {
          const uint64_t mx = desc_mn(base + S::kScores);
#pragma unroll
          for (int p = 1; p >= 0; --p)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16(tbase + 64, kq + k * 2, mx + p * 512 + 128 * k, umma_idesc_bf16_f32(64, 64, false, true), p == 0 || k > 0);
        }
        umma_commit(s_done);
      }
      __syncwarp();
    }
    if (update) {  // ---- keys decayed to the chunk's end, in bf16 parts
#pragma unroll
      for (int u = 0; u < kPasses; ++u) {
        const int r = r0 + kRows * u;
        const uint4 raw = *reinterpret_cast<const uint4*>(smem + (tk - base) + at0 + u * kRows * 128);
        const uint32_t kw[4] = {raw.x, raw.y, raw.z, raw.w};
        const bool there = r >= lo && r < hi;
        const float w = R.kv * pw[there ? (rev ? n_tok - 63 + r : n_tok - 1 - r) : 0];
        uint32_t p0[4], p1[4], p2[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float x = there ? bf_lo(kw[q]) * w : 0.f, y = there ? bf_hi(kw[q]) * w : 0.f;
          p0[q] = bf2(x, y);
          const float x1 = x - bf_lo(p0[q]), y1 = y - bf_hi(p0[q]);
          p1[q] = bf2(x1, y1);
          p2[q] = bf2(x1 - bf_lo(p1[q]), y1 - bf_hi(p1[q]));
        }
        unsigned char* dst = smem + S::kKeys + at0 + u * kRows * 128;
        *reinterpret_cast<uint4*>(dst) = make_uint4(p0[0], p0[1], p0[2], p0[3]);
        *reinterpret_cast<uint4*>(dst + S::kTile) = make_uint4(p1[0], p1[1], p1[2], p1[3]);
        *reinterpret_cast<uint4*>(dst + 2 * S::kTile) = make_uint4(p2[0], p2[1], p2[2], p2[3]);
      }
    }
    if (n_tok < kChunk && a.lengths) {  // rows of v behind the last token may hold anything: P and K' are zero there
#pragma unroll
      for (int u = 0; u < kPasses; ++u) {
        const int r = r0 + kRows * u;
        if (r < lo || r >= hi)
          *reinterpret_cast<uint4*>(smem + (tv - base) + at0 + u * kRows * 128) = make_uint4(0, 0, 0, 0);
      }
    }
    if constexpr (!STATES && D == 128) {
      if (have) {  // ---- the state as an operand: two bf16 parts
#pragma unroll
        for (int n = 0; n < kX; n += 32) {
          uint32_t hi_[16], lo_[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = X[n + 2 * e], y = X[n + 2 * e + 1];
            hi_[e] = bf2(x, y);
            lo_[e] = bf2(x - bf_lo(hi_[e]), y - bf_hi(hi_[e]));
          }
          tmem_st_x16(lanes + half * 32 + n / 2, hi_);
          tmem_st_x16(lanes + 64 + half * 32 + n / 2, lo_);
        }
        tmem_st_wait();
      }
    }
    if constexpr (!STATES) {
      // ---- P: 16 query rows and 32 key columns per warp, up to the diagonal
      if (!wait_phase(s_done, c & 1, lane)) give_up();
      tc_fence_after();
      uint32_t sc[16], o[16];
      const bool some = rev ? half * 2 + 1 >= quarter : half * 2 <= quarter, scaled = D == 64 && have;
      if (some) tmem_ld_frag(lanes + (D == 64 ? 0 : 128) + half * 32, sc);
      if (scaled) tmem_ld_frag(lanes + 64 + half * 32, o);
      tmem_ld_wait();
      if (scaled) {  // Q X -> inter lam^(i + shift) Q X, in place
        const float f0 = R.inter * pw[rev ? 63 - xr : xr + 1], f1 = R.inter * pw[rev ? 55 - xr : xr + 9];
#pragma unroll
        for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * (n & 2 ? f1 : f0));
        tmem_st_frag(lanes + 64 + half * 32, o);
      }
      // the part of the power that belongs to this thread's four key columns inside a block of 16
      const int c0 = rev ? xc : 15 - xc, cs = rev ? 1 : -1;
      const float cf[4] = {pw[c0], pw[c0 + cs], pw[c0 + 8 * cs], pw[c0 + 9 * cs]};
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int kb = half * 2 + m;
        float P[2][4];
        if (kb == quarter) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int ahead = (lane >> 2) + (e >> 1) * 8 - (n * 8 + xc + (e & 1)), gap = rev ? -ahead : ahead;
              P[n][e] = gap >= 0 ? __uint_as_float(sc[m * 8 + n * 4 + e]) * (R.intra * pw[max(gap, 0)]) : 0.f;
            }
        } else if ((kb < quarter) != rev) {
          const int e0 = rev ? kb * 16 - xr : xr - kb * 16 - 15;
          const float f0 = R.intra * pw[e0], f1 = R.intra * pw[rev ? e0 - 8 : e0 + 8];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t* v = sc + m * 8 + n * 4;
            P[n][0] = __uint_as_float(v[0]) * (f0 * cf[2 * n]), P[n][1] = __uint_as_float(v[1]) * (f0 * cf[2 * n + 1]);
            P[n][2] = __uint_as_float(v[2]) * (f1 * cf[2 * n]), P[n][3] = __uint_as_float(v[3]) * (f1 * cf[2 * n + 1]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 2; ++n) P[n][0] = P[n][1] = P[n][2] = P[n][3] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float u = P[n][2 * p], v = P[n][2 * p + 1];
            const uint32_t hi_ = bf2(u, v), lo_ = bf2(u - bf_lo(hi_), v - bf_hi(hi_));
            unsigned char* at = smem + S::kScores + tile_at(xr + 8 * p, 2 * kb + n) + xc * 2;
            *reinterpret_cast<uint32_t*>(at) = hi_;
            *reinterpret_cast<uint32_t*>(at + 8192) = lo_;
          }
      }
      if (D == 64) tmem_st_wait();
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    const bool more = c + S::kStages < nchunks;
    if (ctl) {
      tc_fence_after();
      const uint64_t mv = desc_mn(tv);
      if constexpr (!STATES) {
        if (D == 128 && have) {
          const uint64_t kq = umma_desc_sw128_kmajor(tq);
#pragma unroll
          for (int p = 1; p >= 0; --p)
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              umma_ts(tbase + 192, tbase + p * 64 + k * 8, kq + (k >> 2) * 512 + (k & 3) * 2, umma_idesc_bf16_f32(D, 64),
                      p == 0 || k > 0);
        }
        const uint64_t kp = umma_desc_sw128_kmajor(base + S::kScores);
#pragma unroll
        for (int p = 1; p >= 0; --p)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t acc = p == 0 || k > 0;
            if constexpr (D == 64)
              umma_f16(tbase + 64, kp + p * 512 + k * 2, mv + 128 * k, umma_idesc_bf16_f32(64, 64, false, true), acc || have);
            else
              umma_f16(tbase + 128, mv + 128 * k, kp + p * 512 + k * 2, umma_idesc_bf16_f32(D, 64, true, false), acc);
          }
      }
      if (update) {  // D = 128: behind the products that read X^T, whose columns U takes
        const uint64_t mk = desc_mn(base + S::kKeys);
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t part = mk + p * (S::kTile >> 4) + 128 * k;
            umma_f16(tbase, D == 64 ? part : mv + 128 * k, D == 64 ? mv + 128 * k : part,
                     umma_idesc_bf16_f32(D, D, true, true), p < 2 || k > 0);
          }
      }
      umma_commit(done);
      if (!STATES && D == 64 && more) load(c + 1, 0, 2);  // nothing reads q and k any more
    }
    __syncwarp();
    if (!wait_phase(done, c & 1, lane)) give_up();
    tc_fence_after();
    if (ctl && more) load(c + S::kStages, !STATES && D == 64 ? 2 : 0, S::kTiles);
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
          float s0 = X[n + e], s1 = X[n + e + 1];
          fma2(s0, s1, rest, __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
          fma2(X[n + e], X[n + e + 1], keep, s0, s1);
        }
      }
    }
    if constexpr (!STATES) {
      // ---- the output, through the keys' space so that whole 16-byte groups are stored
      unsigned char* o_tile = smem + S::kKeys;
      __nv_bfloat16* out = R.out + b * R.ob + h * R.oh + (long long)first_row(c) * R.ot;
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
          if (r >= lo && r < hi)
            *reinterpret_cast<uint4*>(out + r * R.ot + g * 8) = *reinterpret_cast<const uint4*>(o_tile + tile_at(r, g));
        }
      } else {
        // fragments of 16 value rows x 8 tokens, stored transposed
        float f[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int r = half * 32 + (n >> 1) * 8 + xc + (n & 1);
          f[n] = have ? R.inter * pw[rev ? 63 - r : r + 1] : 0.f;
        }
#pragma unroll
        for (int hl = 0; hl < 2; ++hl) {
          const uint32_t from = lanes + ((uint32_t)(hl * 16) << 16) + 128 + half * 32;
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
#pragma unroll
        for (int u = 0; u < kPasses; ++u) {
          const int r = r0 + kRows * u;
          if (r >= lo && r < hi)
            *reinterpret_cast<uint4*>(out + r * R.ot + g0 * 8) =
                *reinterpret_cast<const uint4*>(o_tile + at0 + u * kRows * 128);
        }
      }
      have = true;
    }
    tc_fence_before();
  }

  if constexpr (!STATES) {
    // rows of the batch that hold no token (index >= length) give zeros
    __nv_bfloat16* rows = R.out + b * R.ob + h * R.oh;
    const int from = max(t_begin, min(len, t_end));
    for (int e = tid; e < (t_end - from) * kGroups; e += S::kThreads)
      *reinterpret_cast<uint4*>(rows + (long long)(from + e / kGroups) * R.ot + (e % kGroups) * 8) = make_uint4(0, 0, 0, 0);
  }
  if (want_final) {
    float* dst = STATES ? R.segments + ((size_t)bh * a.nseg + seg) * D * D : R.final_state + (size_t)bh * D * D;
#pragma unroll
    for (int n = 0; n < kX; ++n) dst[x_at(n)] = X[n];
  }
  for (int c = seen; c < min(nchunks, seen + S::kStages); ++c)  // no load may still be landing when the block exits
    wait_phase(full + (S::kStages == 2 ? c & 1 : 0), (S::kStages == 2 ? c >> 1 : c) & 1, lane);
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
  if (R.segments_from >= 0) return;  // reads another role's segments
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
// place and sums its part of q^T S; bound by reading and writing the state.
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
cudaError_t launch_chunks(const DecayArgs& a, const DecayMaps& maps, int roles, cudaStream_t s) {
  using S = Shape<D, STATES>;
  const cudaError_t e =
      cudaFuncSetAttribute(k_decay_chunk<D, STATES>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  k_decay_chunk<D, STATES><<<dim3(a.B * a.H, a.nseg, roles), S::kThreads, S::kSmem, s>>>(a, maps);
  return cudaGetLastError();
}

template <int D> cudaError_t decay_typed(const DecayArgs& a, cudaStream_t s, int* launches) {
  *launches = 0;
  DecayMaps maps;
  for (int i = 0; i < a.nin; ++i) {
    const DecayInput& t = a.in[i];
    const cudaError_t e = make_tmap_bf16_heads(&maps.in[i], t.p, a.B, a.T, a.H, D, t.sb, t.st, t.sh);
    if (e != cudaSuccess) return e;
  }
  if (a.nseg > 1) {
    // roles that read another role's segment states come last and need no states of their own
    int own = 0;
    while (own < a.nroles && a.role[own].segments_from < 0) ++own;
    const cudaError_t e = launch_chunks<D, true>(a, maps, own, s);
    if (e != cudaSuccess) return e;
    k_decay_scan<D><<<dim3(a.B * a.H, D * D / 1024, own), 256, 0, s>>>(a);
    *launches += 2;
  }
  *launches += 1;
  return launch_chunks<D, false>(a, maps, a.nroles, s);
}
}  // namespace

unsigned int decay_error_flag() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_decay_error, sizeof(v));
  return v;
}

// Two blocks per SM are resident. Whole sequences take `chunks` steps of a block,
// n segments ceil(chunks / n) of the main kernel and of the state-only one, and two
// more launches. In units of a main step with two blocks on the SM (3.3 us for D =
// 64, 4.5 us for D = 128): a step of a block that has the SM to itself 0.75, a
// state-only step 0.65, the two launches 2.5 (measured at B H = 96, T = 1024, D =
// 64: 38 us whole, 42 us in 3 segments; at 16 heads of 128 and T = 16385, 18
// segments take 152 us).
int decay_segments(int B, int T, int H, int D, int roles) {
  const int chunks = (T + kChunk - 1) / kChunk;
  const long long blocks = (long long)B * H * roles, slots = 148LL * 2;
  const auto steps = [&](long long n) { return (double)((chunks + n - 1) / n); };
  if (blocks * 2 > slots) return 1;
  const long long n = slots / blocks < chunks ? slots / blocks : chunks;
  const double whole = chunks * (blocks <= 148 ? 0.75 : 1.0), split = steps(n) * 1.65 + 2.5;
  return split < whole ? (int)n : 1;
}

cudaError_t decay_attention(const DecayArgs& a, cudaStream_t s, int* launches) {
  if (a.nroles < 1 || a.nroles > 3 || a.nin < 1 || a.nin > 4 || a.B < 1 || a.H < 1 || a.T < 1 || (long long)a.B * a.H > 0x7fffffffLL || a.nseg > 65535 || a.nseg < 1 ||
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
