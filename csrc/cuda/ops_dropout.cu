// Dropout from a counter-based generator (sm_100a), alone and inside the
// residual add + LayerNorm of a decoder block. No mask is stored: the backward
// pass draws the same numbers again.
//
// Draws: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", 2011). Block b of 8 consecutive elements takes the
// counter (b low, b high, site, step) under the key (seed low, seed high); its
// 128 bits are eight 16-bit draws, the low half of each word first. An element
// is kept when its draw is >= threshold = p * 65536 rounded to a whole number,
// and multiplied by 65536 / (65536 - threshold), the inverse of the exact
// probability to be kept. 16 bits per draw instead of 32 halve the generator's
// share: ten rounds are about 60 integer instructions per 8 elements, and the
// multiplier is busy about as long as the memory (4 bytes per element). Measured:
// 64 Mi bf16 elements in 48 us, 5.6 TB/s.
//
// (seed, step) are read from device memory, so a captured graph draws anew when
// the step advances between replays; the forward kernel notes the two values it
// used, and the backward reads those.
#include "decoder_api.h"
#include "pack.cuh"
#include "sm100.cuh"

namespace nexar {
using sm100::smem_u32;

namespace {
constexpr int kDropThreads = 256;

// The generator under one (seed, step, site): the ten round keys are formed
// once per thread and stay in registers.
struct Draws {
  uint32_t k0[10], k1[10], site, step;
  NEXAR_D Draws(const int64_t* state, uint32_t site_) : site(site_) {
    const unsigned long long seed = (unsigned long long)state[0];
    step = (uint32_t)(unsigned long long)state[1];
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      k0[r] = (uint32_t)seed + r * 0x9E3779B9u;
      k1[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
      asm volatile("" : "+r"(k0[r]), "+r"(k1[r]));  // kept: formed again per block they cost 20 of 130 instructions
    }
  }
  // The 128 bits of one block.
  NEXAR_D uint4 operator()(unsigned long long block) const {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = site, c3 = step;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u;
      const unsigned long long p1 = (unsigned long long)c2 * 0xCD9E8D57u;
      c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0[r];
      c1 = (uint32_t)p1;
      c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1[r];
      c3 = (uint32_t)p0;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

// Packed fp32 pairs: half the instructions of the scalar forms.
NEXAR_D float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
NEXAR_D float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
NEXAR_D float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
NEXAR_D float2 both(float v) { return make_float2(v, v); }
NEXAR_D void unpack_pairs(const uint4& r, float2* f) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = make_float2(__uint_as_float(u[e] << 16), __uint_as_float(u[e] & 0xffff0000u));
}
NEXAR_D void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // zero-filled where there is no row
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// v[e] = kept ? v[e] * scale : 0 for the block's 8 elements (selected, not
// multiplied by 0: a dropped infinity leaves no NaN). The draws are compared
// where they lie: a word is >= threshold << 16 exactly when its high half is >=
// threshold, and so is the word moved up by 16 for its low half. `below` is
// (threshold << 16) - 1, which fits 32 bits for thresholds 1 .. 65536.
NEXAR_D void drop8(float2* v, const uint4& w, uint32_t below, float scale) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = mul2(v[e], both(scale));
    v[e].x = (u[e] << 16) > below ? v[e].x : 0.f;
    v[e].y = u[e] > below ? v[e].y : 0.f;
  }
}

// U blocks of 8 elements per thread, all loaded before the first is drawn for.
template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kDropThreads) k_dropout(const T* __restrict__ x, T* __restrict__ y, long long n,
                                                          const int64_t* __restrict__ state, uint32_t site,
                                                          uint32_t threshold, float scale,
                                                          int64_t* __restrict__ snapshot) {
  const uint32_t below = (threshold << 16) - 1;
  if (snapshot && blockIdx.x == 0 && threadIdx.x < 2) snapshot[threadIdx.x] = state[threadIdx.x];
  const long long blocks = (n + 7) / 8, first = blockIdx.x * (long long)(U * kDropThreads) + threadIdx.x;
  Pack<T, 8> v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const long long i = first + k * kDropThreads;
    if (VEC && i * 8 + 8 <= n) {
      v[k].load(x + i * 8);
    } else {  // the last block of fewer than 8 elements, or any of them without alignment
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[k].set(e, i * 8 + 2 * e < n ? to_acc<float>(x[i * 8 + 2 * e]) : 0.f,
                 i * 8 + 2 * e + 1 < n ? to_acc<float>(x[i * 8 + 2 * e + 1]) : 0.f);
    }
  }
  const Draws draws(state, site);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const long long i = first + k * kDropThreads;
    if (i >= blocks) return;
    float2 f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = v[k].get(e);
    drop8(f, draws((unsigned long long)i), below, scale);
    if (VEC && i * 8 + 8 <= n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k].set(e, f[e].x, f[e].y);
      v[k].store(y + i * 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i * 8 + e < n) y[i * 8 + e] = from_acc<T, float>(e & 1 ? f[e / 2].y : f[e / 2].x);
    }
  }
}

// ---------------------------------------------------------------- residual add + dropout + LayerNorm
constexpr int kRowWarps = 8;

NEXAR_D float row_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
NEXAR_D uint4 pack_pairs(const float2* f) {
  uint4 r;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __float22bfloat162_rn(f[k]);
  return r;
}

NEXAR_D uint4 stream16(const __nv_bfloat16* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }

// RW warps per row, NP packs of 8 columns per lane; rows of more than 1024 columns
// take two warps, which leaves registers for twice the rows in flight (32768 x 2048:
// 91 us, 5.9 TB/s, against 101 with one warp; 8192 x 768, one warp: 10.8 us). The sum
// is rounded to the stored bf16 before the statistics, as in the operator without
// dropout.
template <int NP, int RW>
__global__ void __launch_bounds__(kRowWarps * 32) k_dropout_ln_fwd(
    const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ r, const __nv_bfloat16* __restrict__ rb,
    __nv_bfloat16* __restrict__ sum_out, const __nv_bfloat16* __restrict__ w, const __nv_bfloat16* __restrict__ b,
    __nv_bfloat16* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int R, int C, float eps,
    const int64_t* __restrict__ state, uint32_t site, uint32_t threshold, float scale,
    int64_t* __restrict__ snapshot) {
  if (blockIdx.x == 0 && threadIdx.x < 2) snapshot[threadIdx.x] = state[threadIdx.x];
  const int lane = threadIdx.x & (32 * RW - 1), slot = threadIdx.x / (32 * RW);
  const int row = blockIdx.x * (kRowWarps / RW) + slot;
  if (row >= R) return;  // all warps of the row
  __shared__ float red[2][kRowWarps];
  auto row_total = [&](float v, int which) {
    v = row_sum(v);
    if constexpr (RW == 2) {
      const int warp = threadIdx.x >> 5;
      if ((threadIdx.x & 31) == 0) red[which][warp] = v;
      asm volatile("bar.sync %0, 64;" ::"r"(slot + 1) : "memory");
      v = red[which][warp & ~1] + red[which][warp | 1];  // the same order in both warps
    }
    return v;
  };
  const Draws draws(state, site);
  const uint32_t below = (threshold << 16) - 1;
  const size_t base = (size_t)row * C;
  uint4 vx[NP], vr[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int col = (lane + 32 * RW * k) * 8;
    if (col < C) {
      vx[k] = stream16(x + base + col);
      vr[k] = stream16(r + base + col);
    }
  }
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int col = (lane + 32 * RW * k) * 8;
    if (col < C) {
      float2 a[4], d[4];
      unpack_pairs(vx[k], a);
      unpack_pairs(vr[k], d);
      if (rb) {
        float2 t[4];
        unpack_pairs(*reinterpret_cast<const uint4*>(rb + col), t);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = add2(d[e], t[e]);
      }
      drop8(d, draws((base + col) >> 3), below, scale);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = add2(a[e], d[e]);
      vx[k] = pack_pairs(a);
      *reinterpret_cast<uint4*>(sum_out + base + col) = vx[k];
      unpack_pairs(vx[k], a);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = add2(s, a[e]);
    }
  }
  const float mu = row_total(s.x + s.y, 0) / C;
  float2 q = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    if ((lane + 32 * RW * k) * 8 < C) {
      float2 a[4];
      unpack_pairs(vx[k], a);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = add2(a[e], both(-mu));
        q = fma2(a[e], a[e], q);
      }
    }
  }
  const float rs = rsqrtf(row_total(q.x + q.y, 1) / C + eps);
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int col = (lane + 32 * RW * k) * 8;
    if (col < C) {
      float2 a[4], wf[4], bf[4];
      unpack_pairs(vx[k], a);
      unpack_pairs(*reinterpret_cast<const uint4*>(w + col), wf);
      unpack_pairs(*reinterpret_cast<const uint4*>(b + col), bf);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = fma2(mul2(add2(a[e], both(-mu)), both(rs)), wf[e], bf[e]);
      *reinterpret_cast<uint4*>(y + base + col) = pack_pairs(a);
    }
  }
  if (lane == 0) {
    mean[row] = mu;
    rstd[row] = rs;
  }
}

// Backward. A block of C/8 threads (whole warps) walks over its rows two at a
// time; a thread owns 8 columns, so the column sums (dw, db, drb) stay in 24
// registers however wide the row is. Each pair of rows costs one barrier
// for the two row sums. The rows come by cp.async, two pairs ahead, each thread
// its own 16 bytes of each: no register holds them on the way, nobody waits for
// another thread's. The blocks' column sums go to `part` and are added in a
// fixed order by k_dropout_ln_columns: no atomics, the same bits every run.
// The normalised value is (x - mean) rstd, as in the forward pass: x rstd - mean rstd
// in one FMA would round mean rstd, which is far from 0 where x is the mean.
// Measured with the columns: 32768 x 2048 in 117 us (671 MB, 5.7 TB/s), 8192 x 768
// in 18. Through registers it took 155 and 23 (one pair ahead at most); three or
// four blocks an SM, or one more stage, take 121 to 127.
constexpr int kBwdRows = 2, kBwdStages = 3;
template <bool BIAS>
__global__ void __launch_bounds__(256, 2) k_dropout_ln_bwd(
    const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ s, const float* __restrict__ mean,
    const float* __restrict__ rstd, const __nv_bfloat16* __restrict__ w, const __nv_bfloat16* __restrict__ dres,
    __nv_bfloat16* __restrict__ dx, __nv_bfloat16* __restrict__ dr, float* __restrict__ part, int R, int C,
    const int64_t* __restrict__ state, uint32_t site, uint32_t threshold, float scale) {
  extern __shared__ __align__(16) uint4 ring[];  // [stage][row][dy, s, dres][thread]
  __shared__ float4 red[2][8];                   // two buffers: one barrier per pair of rows
  const int tid = threadIdx.x, threads = blockDim.x, col = tid * 8;
  const bool mine = col < C;
  const int lane = tid & 31, warp = tid >> 5;
  const Draws draws(state, site);
  const uint32_t below = (threshold << 16) - 1;
  float2 aw[4], ab[4], ad[4], wf[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) aw[e] = ab[e] = ad[e] = wf[e] = make_float2(0.f, 0.f);
  if (mine) unpack_pairs(*reinterpret_cast<const uint4*>(w + col), wf);
  if (tid < 16) red[tid >> 3][tid & 7] = make_float4(0.f, 0.f, 0.f, 0.f);  // warps that a narrow row does not have
  __syncthreads();
  const int stride = gridDim.x * kBwdRows;
  auto slot = [&](int stage, int k, int which) { return ((stage * kBwdRows + k) * 3 + which) * threads + tid; };
  auto prefetch = [&](int row, int stage) {
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) {
      const bool ok = mine && row + k < R;
      const size_t off = ok ? (size_t)(row + k) * C + col : 0;
      cp_async16(smem_u32(ring + slot(stage, k, 0)), dy + off, ok);
      cp_async16(smem_u32(ring + slot(stage, k, 1)), s + off, ok);
      cp_async16(smem_u32(ring + slot(stage, k, 2)), dres ? dres + off : s, ok && dres);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int first = blockIdx.x * kBwdRows;
#pragma unroll
  for (int i = 0; i + 1 < kBwdStages; ++i) prefetch(first + i * stride, i);
  float mu_next[kBwdRows], rs_next[kBwdRows];
  auto load_stats = [&](int row) {
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) {
      const bool ok = row + k < R;
      mu_next[k] = ok ? mean[row + k] : 0.f;
      rs_next[k] = ok ? rstd[row + k] : 0.f;  // rows that are not there: all zero from here on
    }
  };
  load_stats(first);
  const float inv = 1.f / C;
  int buf = 0, stage = 0;
  for (int row0 = first; row0 < R; row0 += stride, buf ^= 1) {
    float mu[kBwdRows], rs[kBwdRows], sums[4];
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) mu[k] = mu_next[k], rs[k] = rs_next[k];
    asm volatile("cp.async.wait_group %0;" ::"n"(kBwdStages - 2) : "memory");
    prefetch(row0 + (kBwdStages - 1) * stride, stage == 0 ? kBwdStages - 1 : stage - 1);
    load_stats(row0 + stride);
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) {
      float2 g[4], x[4], s1 = make_float2(0.f, 0.f), s2 = s1;
      unpack_pairs(ring[slot(stage, k, 0)], g);
      unpack_pairs(ring[slot(stage, k, 1)], x);
      const float2 r2 = both(rs[k]), m2 = both(-mu[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 xh = mul2(add2(x[e], m2), r2), gw = mul2(g[e], wf[e]);
        aw[e] = fma2(g[e], xh, aw[e]);
        ab[e] = add2(ab[e], g[e]);
        s1 = add2(s1, gw);
        s2 = fma2(gw, xh, s2);
      }
      sums[2 * k] = s1.x + s1.y;
      sums[2 * k + 1] = s2.x + s2.y;
    }
    {  // the warp's four sums: lanes 8 i .. 8 i + 7 end with number i
      const bool hi = lane & 16, odd = lane & 8;
      const float a = (hi ? sums[2] : sums[0]) + __shfl_xor_sync(0xffffffffu, hi ? sums[0] : sums[2], 16);
      const float b = (hi ? sums[3] : sums[1]) + __shfl_xor_sync(0xffffffffu, hi ? sums[1] : sums[3], 16);
      float v = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if ((lane & 7) == 0) reinterpret_cast<float*>(&red[buf][warp])[lane >> 3] = v;
    }
    __syncthreads();
    float4 t = red[buf][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      const float4 v = red[buf][i];
      t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
    sums[0] = t.x, sums[1] = t.y, sums[2] = t.z, sums[3] = t.w;
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) {
      float2 g[4], x[4], o[4];
      unpack_pairs(ring[slot(stage, k, 0)], g);
      unpack_pairs(ring[slot(stage, k, 1)], x);
      unpack_pairs(ring[slot(stage, k, 2)], o);
      const float2 r2 = both(rs[k]), m2 = both(-mu[k]);
      const float2 c1 = both(-sums[2 * k] * inv), c2 = both(-sums[2 * k + 1] * inv * rs[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fma2(r2, fma2(g[e], wf[e], fma2(add2(x[e], m2), c2, c1)), o[e]);
      const size_t off = (size_t)(row0 + k) * C + col;
      const uint4 ox = pack_pairs(o);
      drop8(o, draws(off >> 3), below, scale);
      if constexpr (BIAS) {
#pragma unroll
        for (int e = 0; e < 4; ++e) ad[e] = add2(ad[e], o[e]);  // before the rounding of dr
      }
      if (mine && row0 + k < R) {
        *reinterpret_cast<uint4*>(dx + off) = ox;
        *reinterpret_cast<uint4*>(dr + off) = pack_pairs(o);
      }
    }
    stage = stage == kBwdStages - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (mine) {
    float4* p = reinterpret_cast<float4*>(part + (size_t)blockIdx.x * (BIAS ? 3 : 2) * C + col);
    const int c4 = C / 4;
    p[0] = make_float4(aw[0].x, aw[0].y, aw[1].x, aw[1].y);
    p[1] = make_float4(aw[2].x, aw[2].y, aw[3].x, aw[3].y);
    p[c4] = make_float4(ab[0].x, ab[0].y, ab[1].x, ab[1].y);
    p[c4 + 1] = make_float4(ab[2].x, ab[2].y, ab[3].x, ab[3].y);
    if constexpr (BIAS) {
      p[2 * c4] = make_float4(ad[0].x, ad[0].y, ad[1].x, ad[1].y);
      p[2 * c4 + 1] = make_float4(ad[2].x, ad[2].y, ad[3].x, ad[3].y);
    }
  }
}

// Column sums of the P partial rows of W = (2 or 3) C values, in a fixed order:
// 4 lanes of 4 columns by 64 slices of the partial rows per block.
__global__ void __launch_bounds__(256) k_dropout_ln_columns(const float* __restrict__ part, int P, int W, int C,
                                                            __nv_bfloat16* dw, __nv_bfloat16* db,
                                                            __nv_bfloat16* drb) {
  __shared__ float4 red[64][4];
  const int cg = threadIdx.x & 3, sl = threadIdx.x >> 2;
  const int col = (blockIdx.x * 4 + cg) * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < W) {
#pragma unroll 8
    for (int p = sl; p < P; p += 64) {
      const float4 v = *reinterpret_cast<const float4*>(part + (size_t)p * W + col);
      a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
  }
  red[sl][cg] = a;
  __syncthreads();
  if (threadIdx.x < 16) {  // one thread per column
    const int c1 = blockIdx.x * 16 + threadIdx.x;
    if (c1 < W) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < 64; ++j) t += reinterpret_cast<const float*>(red[j])[threadIdx.x];
      const int which = c1 / C;
      (which == 0 ? dw : which == 1 ? db : drb)[c1 % C] = __float2bfloat16_rn(t);
    }
  }
}

// Blocks of the backward: enough rows per block that its partial sums (12 C
// bytes) stay small beside the rows (10 C bytes each), at most the number that
// fits the GPU at once.
int bwd_blocks(int R, int C) {
  const int threads = (C / 8 + 31) / 32 * 32;
  const int per_sm = threads <= 128 ? 4 : 2;
  const int groups = (R + kBwdRows - 1) / kBwdRows;
  return groups < 148 * per_sm ? (groups < 1 ? 1 : groups) : 148 * per_sm;
}

template <typename T>
cudaError_t dropout_typed(const void* x, void* y, long long n, const int64_t* state, uint32_t site, uint32_t thr,
                          float scale, int64_t* snapshot, cudaStream_t s) {
  const long long blocks = (n + 7) / 8;
  const T* xi = reinterpret_cast<const T*>(x);
  T* yo = reinterpret_cast<T*>(y);
  constexpr int U = sizeof(T) == 4 ? 2 : 4;
  const bool many = blocks > 148LL * 2048;  // else one block per thread, for the shortest path
  const long long per = (many ? U : 1) * kDropThreads, grid = (blocks + per - 1) / per;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  const auto kernel = (uintptr_t)x % 16 || (uintptr_t)y % 16 ? (many ? k_dropout<T, false, U> : k_dropout<T, false, 1>)
                                                             : (many ? k_dropout<T, true, U> : k_dropout<T, true, 1>);
  kernel<<<(unsigned)grid, kDropThreads, 0, s>>>(xi, yo, n, state, site, thr, scale, snapshot);
  return cudaGetLastError();
}
}  // namespace

cudaError_t dropout(const void* x, void* y, long long n, int dtype, const int64_t* state, uint32_t site,
                    uint32_t threshold, float scale, int64_t* snapshot, cudaStream_t s) {
  if (n <= 0 || threshold < 1 || threshold > 65536) return cudaErrorInvalidValue;
  if (dtype == 0) return dropout_typed<__nv_bfloat16>(x, y, n, state, site, threshold, scale, snapshot, s);
  if (dtype == 1) return dropout_typed<__half>(x, y, n, state, site, threshold, scale, snapshot, s);
  return dropout_typed<float>(x, y, n, state, site, threshold, scale, snapshot, s);
}

cudaError_t dropout_ln_fwd(const __nv_bfloat16* x, const __nv_bfloat16* r, const __nv_bfloat16* rb,
                           __nv_bfloat16* sum_out, const __nv_bfloat16* w, const __nv_bfloat16* b, __nv_bfloat16* y,
                           float* mean, float* rstd, int R, int C, float eps, const int64_t* state, uint32_t site,
                           uint32_t threshold, float scale, int64_t* snapshot, cudaStream_t s) {
  if (C % 8 || C > 2048 || R < 1 || threshold < 1 || threshold > 65536) return cudaErrorInvalidValue;
#define NEXAR_DROP_FWD(NP, RW)                                                                              \
  k_dropout_ln_fwd<NP, RW><<<(R + kRowWarps / RW - 1) / (kRowWarps / RW), kRowWarps * 32, 0, s>>>(            \
      x, r, rb, sum_out, w, b, y, mean, rstd, R, C, eps, state, site, threshold, scale, snapshot)
  if (C <= 256) NEXAR_DROP_FWD(1, 1);
  else if (C <= 512) NEXAR_DROP_FWD(2, 1);
  else if (C <= 768) NEXAR_DROP_FWD(3, 1);
  else if (C <= 1024) NEXAR_DROP_FWD(4, 1);
  else if (C <= 1536) NEXAR_DROP_FWD(3, 2);
  else NEXAR_DROP_FWD(4, 2);
#undef NEXAR_DROP_FWD
  return cudaGetLastError();
}

size_t dropout_ln_bwd_scratch_floats(int R, int C) { return (size_t)bwd_blocks(R, C) * 3 * C; }

cudaError_t dropout_ln_bwd(const __nv_bfloat16* dy, const __nv_bfloat16* s_in, const float* mean, const float* rstd,
                           const __nv_bfloat16* w, const __nv_bfloat16* dres, __nv_bfloat16* dx, __nv_bfloat16* dr,
                           __nv_bfloat16* dw, __nv_bfloat16* db, __nv_bfloat16* drb, float* scratch, int R, int C,
                           const int64_t* state, uint32_t site, uint32_t threshold, float scale, cudaStream_t s) {
  if (C % 8 || C > 2048 || R < 1 || threshold < 1 || threshold > 65536) return cudaErrorInvalidValue;
  const int grid = bwd_blocks(R, C), threads = (C / 8 + 31) / 32 * 32;
  const int ring = kBwdStages * kBwdRows * 3 * threads * 16;
  const auto kernel = drb ? k_dropout_ln_bwd<true> : k_dropout_ln_bwd<false>;
  cudaError_t e = cudaSuccess;
  if (ring > 48 * 1024)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBwdStages * kBwdRows * 3 * 256 * 16);
  if (e != cudaSuccess) return e;
  kernel<<<grid, threads, ring, s>>>(dy, s_in, mean, rstd, w, dres, dx, dr, scratch, R, C, state, site, threshold,
                                     scale);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int W = (drb ? 3 : 2) * C;
  k_dropout_ln_columns<<<(W + 15) / 16, 256, 0, s>>>(scratch, grid, W, C, dw, db, drb);
  return cudaGetLastError();
}

}  // namespace nexar
