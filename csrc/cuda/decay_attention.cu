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
// Roundings. Products are bf16 tensor-core products with fp32 sums. The decayed
// keys that enter the state are split into three bf16 parts (24 bits, all of an
// fp32 value), so the state is an fp32 state; scores and states that enter the
// output are split into two parts (16 bits), well below the rounding of the bf16
// output.
#include "common.cuh"
#include "decoder_api.h"

namespace nexar {

namespace {
constexpr int kChunk = 64;

NEXAR_D uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
NEXAR_D void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // zero-filled where there is no token
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
NEXAR_D void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> NEXAR_D void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
NEXAR_D void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
NEXAR_D void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
NEXAR_D void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
NEXAR_D uint32_t bf2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
NEXAR_D float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
NEXAR_D float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// Byte offset of 16-byte group `g` of row `r` in a tile of D bf16 columns; the
// group index is permuted by the row so that ldmatrix finds no bank conflicts.
template <int D> NEXAR_D uint32_t tile_at(int r, int g) { return (uint32_t)(r * D * 2 + ((g ^ (r & 7)) << 4)); }

// Per-thread addresses of ldmatrix.x4 over a 16 x 16 block at (row, col): the
// four 8 x 8 matrices are (rows 0-7, 8-15) x (cols 0-7, 8-15), rows first.
template <int D> NEXAR_D uint32_t block_at(uint32_t tile, int row, int col, int lane) {
  return tile + tile_at<D>(row + (lane & 15), (col >> 3) + (lane >> 4));
}

template <int D> struct Shape {
  static constexpr int kWarps = D / 16;           // one warp per 16 rows of the state
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTile = kChunk * D * 2;    // bytes of one tile of q, k or v
  static constexpr int kState = D * D * 2;        // bytes of one bf16 part of the state
  static constexpr int kSmem = 6 * kTile + 2 * kState + 512;
  static constexpr int kSmemStates = 4 * kTile + 512;  // k and v only, twice
};

template <int D, bool STATES>
__global__ void __launch_bounds__(Shape<D>::kThreads, D == 64 ? (STATES ? 4 : 3) : (STATES ? 2 : 1))
    k_decay_chunk(const __grid_constant__ DecayArgs a) {
  using S = Shape<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  const DecayRole& R = a.role[blockIdx.z];
  const int bh = blockIdx.x, seg = blockIdx.y;
  const int b = bh / a.H, h = bh % a.H;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = a.lengths ? max(0, min(a.lengths[b], a.T)) : a.T;
  const int t_begin = seg * a.seg_tokens;
  const int t_end = min(a.T, t_begin + a.seg_tokens);   // index i, counted from the first token of the direction
  const int live = max(0, min(len, t_end) - t_begin);   // tokens of this segment that exist
  const int nchunks = (live + kChunk - 1) / kChunk;

  constexpr int kTiles = STATES ? 2 : 3;
  unsigned char* tiles = smem;                                   // [2][kTiles][kTile]
  unsigned char* sx = smem + 2 * kTiles * S::kTile;              // [2 parts][D][D] bf16 (not for STATES)
  float* pw = reinterpret_cast<float*>(smem + 2 * kTiles * S::kTile + (STATES ? 0 : 2 * S::kState));  // lam^0 .. lam^64
  const uint32_t tiles_u = smem_addr(tiles), sx_u = smem_addr(sx);

  const double g = (double)a.log_decay[h];
  for (int i = tid; i <= kChunk; i += S::kThreads) pw[i] = i ? (float)exp(g * i) : 1.f;
  // What the rounding of lam^64 leaves out: over hundreds of chunks that error would add up.
  const float full_rest = (float)(exp(g * kChunk) - (double)(float)exp(g * kChunk));

  // Token index i sits at row i, or at len - 1 - i when the direction is reversed.
  auto prefetch = [&](int c) {
    const int i0 = t_begin + c * kChunk;
    const uint32_t dst = tiles_u + (c & 1) * kTiles * S::kTile;
    constexpr int kGroups = D / 8;
#pragma unroll
    for (int w = 0; w < kTiles; ++w) {
      const int which = STATES ? w + 1 : w;
      const __nv_bfloat16* p = which == 0 ? R.q + b * R.qb + h * R.qh
                               : which == 1 ? R.k + b * R.kb + h * R.kh : R.v + b * R.vb + h * R.vh;
      const long long st = which == 0 ? R.qt : which == 1 ? R.kt : R.vt;
#pragma unroll
      for (int u = 0; u < kChunk * kGroups / S::kThreads; ++u) {
        const int e = tid + u * S::kThreads, r = e / kGroups, gq = e % kGroups;
        const int i = i0 + r;
        const bool ok = i < len;
        const long long t = ok ? (R.reverse ? len - 1 - i : i) : 0;
        cp_async16(dst + w * S::kTile + tile_at<D>(r, gq), p + t * st + gq * 8, ok);
      }
    }
    cp_commit();
  };

  // ---- state: warp w holds rows [16 w, 16 w + 16), all D columns, as accumulator fragments
  float X[D / 8][4];
  const int xr = warp * 16 + (lane >> 2), xc = (lane & 3) * 2;
  const float* x0 = nullptr;
  bool x0_t = false;
  if constexpr (!STATES) {
    if (a.nseg > 1) {
      const bool own = R.segments_from < 0;
      const float* base = own ? R.segments : a.role[R.segments_from].segments;
      x0 = base + ((size_t)bh * a.nseg + seg) * D * D;
      x0_t = !own;
    } else if (R.init) {
      x0 = R.init + (size_t)bh * D * D;
      x0_t = R.init_transposed;
    }
  }
  if (nchunks > 0) prefetch(0);
  if (x0) {
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = xr + (e >> 1) * 8, c = n * 8 + xc + (e & 1);
        X[n][e] = x0_t ? x0[c * D + r] : x0[r * D + c];
      }
  } else {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) X[n][0] = X[n][1] = X[n][2] = X[n][3] = 0.f;
  }
  bool have = x0 != nullptr;  // a state that is known to be zero is not multiplied

  auto publish = [&]() {  // bf16 parts of the state for the next chunk's X^T q
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t hi = bf2(X[n][2 * p], X[n][2 * p + 1]);
        const uint32_t lo = bf2(X[n][2 * p] - bf_lo(hi), X[n][2 * p + 1] - bf_hi(hi));
        const uint32_t at = tile_at<D>(xr + 8 * p, n) + xc * 2;
        *reinterpret_cast<uint32_t*>(sx + at) = hi;
        *reinterpret_cast<uint32_t*>(sx + S::kState + at) = lo;
      }
  };
  if constexpr (!STATES) {
    if (have) publish();
  }
  const bool want_final = STATES || (R.final_state != nullptr && a.nseg == 1);
  const int shift = R.reverse ? 0 : 1;  // exponents: i + shift and n - shift - j

  for (int c = 0; c < nchunks; ++c) {
    cp_wait<0>();
    __syncthreads();  // chunk c and the published state are visible; the other buffer is free
    if (c + 1 < nchunks) prefetch(c + 1);
    const int n_tok = min(kChunk, live - c * kChunk);
    const uint32_t buf = tiles_u + (c & 1) * kTiles * S::kTile;
    const uint32_t tq = buf, tk = buf + (STATES ? 0 : S::kTile), tv = tk + S::kTile;
    const bool update = want_final || c + 1 < nchunks;

    [[maybe_unused]] float O[8][4];
    [[maybe_unused]] const int rb = warp & 3, ch = warp >> 2;  // 16 query rows, 64 output columns
    [[maybe_unused]] const bool rows = rb * 16 < n_tok;
    if constexpr (!STATES) {
#pragma unroll
      for (int n = 0; n < 8; ++n) O[n][0] = O[n][1] = O[n][2] = O[n][3] = 0.f;
      if (rows) {
        uint32_t qf[D / 16][4];
#pragma unroll
        for (int k = 0; k < D / 16; ++k) ldsm4(block_at<D>(tq, rb * 16, k * 16, lane), qf[k]);
        const int i_lo = rb * 16 + (lane >> 2);
        if (have) {
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                uint32_t f[4];
                ldsm4t(block_at<D>(sx_u + part * S::kState, k * 16, ch * 64 + n * 16, lane), f);
                mma16816(O[2 * n], qf[k], f[0], f[1]);
                mma16816(O[2 * n + 1], qf[k], f[2], f[3]);
              }
          const float f0 = R.inter * pw[i_lo + shift], f1 = R.inter * pw[i_lo + 8 + shift];
#pragma unroll
          for (int n = 0; n < 8; ++n) O[n][0] *= f0, O[n][1] *= f0, O[n][2] *= f1, O[n][3] *= f1;
        }
        // lam^15-jj of this thread's four key columns inside a block of 16
        const int jc = (lane & 3) * 2;
        const float cf[4] = {pw[15 - jc], pw[14 - jc], pw[7 - jc], pw[6 - jc]};
        for (int kb = 0; kb <= rb; ++kb) {
          float P[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t f[4];
            ldsm4(block_at<D>(tk, kb * 16, k * 16, lane), f);
            mma16816(P[0], qf[k], f[0], f[2]);
            mma16816(P[1], qf[k], f[1], f[3]);
          }
          if (kb < rb) {
            const float r0 = R.intra * pw[i_lo - kb * 16 - 15], r1 = R.intra * pw[i_lo + 8 - kb * 16 - 15];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              P[n][0] *= r0 * cf[2 * n], P[n][1] *= r0 * cf[2 * n + 1];
              P[n][2] *= r1 * cf[2 * n], P[n][3] *= r1 * cf[2 * n + 1];
            }
          } else {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int gap = (lane >> 2) + (e >> 1) * 8 - (n * 8 + jc + (e & 1));
                P[n][e] = gap >= 0 ? P[n][e] * (R.intra * pw[gap]) : 0.f;
              }
          }
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // A fragment: (row, row + 8) x (8 columns, next 8)
            const float u = P[e >> 1][(e & 1) * 2], v = P[e >> 1][(e & 1) * 2 + 1];
            ph[e] = bf2(u, v);
            pl[e] = bf2(u - bf_lo(ph[e]), v - bf_hi(ph[e]));
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            uint32_t f[4];
            ldsm4t(block_at<D>(tv, kb * 16, ch * 64 + n * 16, lane), f);
            mma16816(O[2 * n], ph, f[0], f[1]);
            mma16816(O[2 * n + 1], ph, f[2], f[3]);
            mma16816(O[2 * n], pl, f[0], f[1]);
            mma16816(O[2 * n + 1], pl, f[2], f[3]);
          }
        }
      }
    }

    if (update) {
      // A = k^T: rows are state rows, columns tokens (transposed 16 x 16 blocks of the key tile), decayed to the
      // chunk's end and split into three parts
      const float keep = pw[n_tok], rest = n_tok == kChunk ? full_rest : 0.f;
      uint32_t kh[4][4], km[4][4], kl[4][4];
#pragma unroll
      for (int tb = 0; tb < 4; ++tb) {
        uint32_t kf[4];
        ldsm4t(tk + tile_at<D>(tb * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * warp + ((lane >> 3) & 1)), kf);
        const int j = tb * 16 + (lane & 3) * 2;
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int p = n_tok - shift - (j + (e & 1) + (e >> 1) * 8);  // rows behind the last token are zero
          w[e] = R.kv * pw[max(p, 0)];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = bf_lo(kf[e]) * w[(e >> 1) * 2], v = bf_hi(kf[e]) * w[(e >> 1) * 2 + 1];
          kh[tb][e] = bf2(u, v);
          const float u1 = u - bf_lo(kh[tb][e]), v1 = v - bf_hi(kh[tb][e]);
          km[tb][e] = bf2(u1, v1);
          kl[tb][e] = bf2(u1 - bf_lo(km[tb][e]), v1 - bf_hi(km[tb][e]));
        }
      }
      // The chunk's own sum is formed apart and added once: the tensor cores cut off what does not fit their
      // accumulator, which on a state that grows over thousands of tokens would add up.
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        float U[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        uint32_t f[4][4];
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) ldsm4t(block_at<D>(tv, tb * 16, n * 16, lane), f[tb]);
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
          mma16816(U[0], kl[tb], f[tb][0], f[tb][1]);
          mma16816(U[1], kl[tb], f[tb][2], f[tb][3]);
        }
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
          mma16816(U[0], km[tb], f[tb][0], f[tb][1]);
          mma16816(U[1], km[tb], f[tb][2], f[tb][3]);
        }
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
          mma16816(U[0], kh[tb], f[tb][0], f[tb][1]);
          mma16816(U[1], kh[tb], f[tb][2], f[tb][3]);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            X[2 * n + m][e] = fmaf(X[2 * n + m][e], keep, fmaf(X[2 * n + m][e], rest, U[m][e]));
      }
    }
    if constexpr (!STATES) {
      __syncthreads();  // everyone has read the state's parts and the query tile
      if (update && c + 1 < nchunks) publish();
      have = true;
      if (rows) {  // through the query tile, so that whole 16-byte groups are stored
        unsigned char* o_tile = tiles + (c & 1) * kTiles * S::kTile;
        const int r = rb * 16 + (lane >> 2);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          *reinterpret_cast<uint32_t*>(o_tile + tile_at<D>(r, ch * 8 + n) + xc * 2) = bf2(O[n][0], O[n][1]);
          *reinterpret_cast<uint32_t*>(o_tile + tile_at<D>(r + 8, ch * 8 + n) + xc * 2) = bf2(O[n][2], O[n][3]);
        }
        __syncwarp();
        __nv_bfloat16* out = R.out + b * R.ob + h * R.oh;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int rr = rb * 16 + u * 4 + (lane >> 3), gq = ch * 8 + (lane & 7);
          if (rr < n_tok) {
            const int i = t_begin + c * kChunk + rr;
            const long long t = R.reverse ? len - 1 - i : i;
            *reinterpret_cast<uint4*>(out + t * R.ot + gq * 8) =
                *reinterpret_cast<const uint4*>(o_tile + tile_at<D>(rr, gq));
          }
        }
      }
    }
  }

  if constexpr (!STATES) {
    // rows of the batch that hold no token (index >= length) give zeros
    __nv_bfloat16* out = R.out + b * R.ob + h * R.oh;
    constexpr int kGroups = D / 8;
    for (int e = tid; e < (t_end - max(t_begin, min(len, t_end))) * kGroups; e += S::kThreads) {
      const int i = max(t_begin, min(len, t_end)) + e / kGroups;
      *reinterpret_cast<uint4*>(out + (long long)i * R.ot + (e % kGroups) * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  if (want_final) {
    float* dst = STATES ? R.segments + ((size_t)bh * a.nseg + seg) * D * D : R.final_state + (size_t)bh * D * D;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        *reinterpret_cast<float2*>(dst + (size_t)(xr + 8 * p) * D + n * 8 + xc) = make_float2(X[n][2 * p], X[n][2 * p + 1]);
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
  const double g = (double)a.log_decay[h];
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
  // whole segments, then one with the last tokens, then empty ones
  const int whole = len / a.seg_tokens, rest = len - whole * a.seg_tokens;
  const double whole_decay = exp(g * a.seg_tokens);
  const float full = (float)whole_decay, full_rest = (float)(whole_decay - (double)full);
  const float part = rest ? (float)exp(g * rest) : 1.f;
#pragma unroll 4
  for (int s = 0; s < a.nseg; ++s) {
    const float f = s < whole ? full : (s == whole ? part : 1.f), r = s < whole ? full_rest : 0.f;
    const float4 u = p[(size_t)s * (D * D / 4)];
    p[(size_t)s * (D * D / 4)] = x;
    x.x = fmaf(f, x.x, fmaf(r, x.x, u.x)), x.y = fmaf(f, x.y, fmaf(r, x.y, u.y));
    x.z = fmaf(f, x.z, fmaf(r, x.z, u.z)), x.w = fmaf(f, x.w, fmaf(r, x.w, u.w));
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

template <typename K> cudaError_t allow_smem(K kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int D> cudaError_t decay_typed(const DecayArgs& a, cudaStream_t s, int* launches) {
  using S = Shape<D>;
  *launches = 0;
  if (a.nseg > 1) {
    cudaError_t e = allow_smem(k_decay_chunk<D, true>, S::kSmemStates);
    if (e != cudaSuccess) return e;
    // roles that read another role's segment states come last and need no states of their own
    int own = 0;
    while (own < a.nroles && a.role[own].segments_from < 0) ++own;
    k_decay_chunk<D, true><<<dim3(a.B * a.H, a.nseg, own), S::kThreads, S::kSmemStates, s>>>(a);
    k_decay_scan<D><<<dim3(a.B * a.H, D * D / 1024, own), 256, 0, s>>>(a);
    *launches += 2;
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  cudaError_t e = allow_smem(k_decay_chunk<D, false>, S::kSmem);
  if (e != cudaSuccess) return e;
  k_decay_chunk<D, false><<<dim3(a.B * a.H, a.nseg, a.nroles), S::kThreads, S::kSmem, s>>>(a);
  *launches += 1;
  return cudaGetLastError();
}
}  // namespace

int decay_segments(int B, int T, int H, int D, int roles) {
  // Blocks resident at once: 3 per SM for D = 64, 1 for D = 128.
  const int chunks = (T + kChunk - 1) / kChunk;
  const long long blocks = (long long)B * H * roles, want = 148LL * (D == 64 ? 3 : 1);
  if (blocks * 2 > want || chunks < 4) return 1;
  long long n = (want + blocks - 1) / blocks;
  if (n > chunks / 2) n = chunks / 2;
  return (int)n;
}

cudaError_t decay_attention(const DecayArgs& a, cudaStream_t s, int* launches) {
  if (a.nroles < 1 || a.nroles > 3 || a.B < 1 || a.H < 1 || a.T < 1 || (long long)a.B * a.H > 0x7fffffffLL || a.nseg > 65535 || a.nseg < 1 ||
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
