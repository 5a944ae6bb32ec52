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
// 64 Mi bf16 elements in 49 us, 5.5 TB/s.
//
// (seed, step) are read from device memory, so a captured graph draws anew when
// the step advances between replays; the forward kernel notes the two values it
// used, and the backward reads those.
#include "decoder_api.h"
#include "pack.cuh"

namespace nexar {

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

// v[e] = kept ? v[e] * scale : 0 for the block's 8 elements (selected, not
// multiplied by 0: a dropped infinity leaves no NaN). The draws are compared
// where they lie: a word is >= threshold << 16 exactly when its high half is >=
// threshold, and so is the word moved up by 16 for its low half. `below` is
// (threshold << 16) - 1, which fits 32 bits for thresholds 1 .. 65536.
NEXAR_D void drop8(float* v, const uint4& w, uint32_t below, float scale) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = (u[e] << 16) > below ? v[2 * e] * scale : 0.f;
    v[2 * e + 1] = u[e] > below ? v[2 * e + 1] * scale : 0.f;
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
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 t = v[k].get(e);
      f[2 * e] = t.x, f[2 * e + 1] = t.y;
    }
    drop8(f, draws((unsigned long long)i), below, scale);
    if (VEC && i * 8 + 8 <= n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k].set(e, f[2 * e], f[2 * e + 1]);
      v[k].store(y + i * 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i * 8 + e < n) y[i * 8 + e] = from_acc<T, float>(f[e]);
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
NEXAR_D void unpack8(const uint4& r, float* f) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 t = __bfloat1622float2(h[k]);
    f[2 * k] = t.x;
    f[2 * k + 1] = t.y;
  }
}
NEXAR_D uint4 pack8(const float* f) {
  uint4 r;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
  return r;
}
NEXAR_D uint4 stream16(const __nv_bfloat16* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }

// RW warps per row, NP packs of 8 columns per lane; rows of more than 1024 columns
// take two warps, which leaves registers for twice the rows in flight (32768 x 2048:
// 107 us, 5.0 TB/s, against 122 with one warp; 8192 x 768, one warp: 14 us). The sum
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
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int col = (lane + 32 * RW * k) * 8;
    if (col < C) {
      float a[8], d[8];
      unpack8(vx[k], a);
      unpack8(vr[k], d);
      if (rb) {
        float t[8];
        unpack8(*reinterpret_cast<const uint4*>(rb + col), t);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] += t[e];
      }
      drop8(d, draws((base + col) >> 3), below, scale);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] += d[e];
      vx[k] = pack8(a);
      *reinterpret_cast<uint4*>(sum_out + base + col) = vx[k];
      unpack8(vx[k], a);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += a[e];
    }
  }
  const float mu = row_total(s, 0) / C;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    if ((lane + 32 * RW * k) * 8 < C) {
      float a[8];
      unpack8(vx[k], a);
#pragma unroll
      for (int e = 0; e < 8; ++e) q += (a[e] - mu) * (a[e] - mu);
    }
  }
  const float rs = rsqrtf(row_total(q, 1) / C + eps);
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int col = (lane + 32 * RW * k) * 8;
    if (col < C) {
      float a[8], wf[8], bf[8];
      unpack8(vx[k], a);
      unpack8(*reinterpret_cast<const uint4*>(w + col), wf);
      unpack8(*reinterpret_cast<const uint4*>(b + col), bf);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = (a[e] - mu) * rs * wf[e] + bf[e];
      *reinterpret_cast<uint4*>(y + base + col) = pack8(a);
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
// for the two row sums. The blocks' column sums go to `part` and are added in a
// fixed order by k_dropout_ln_columns: no atomics, the same bits every run.
// Measured: 32768 x 2048 in 149 us (671 MB, 4.5 TB/s) and 4 us for the columns; 8192
// x 768 in 15 and 5 us. 16 warps an SM issue in 58 % of the cycles, a third of that
// for the draws; one or four rows at a time, or half the block, took longer.
constexpr int kBwdRows = 2;
template <bool BIAS>
__global__ void __launch_bounds__(256, 2) k_dropout_ln_bwd(
    const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ s, const float* __restrict__ mean,
    const float* __restrict__ rstd, const __nv_bfloat16* __restrict__ w, const __nv_bfloat16* __restrict__ dres,
    __nv_bfloat16* __restrict__ dx, __nv_bfloat16* __restrict__ dr, float* __restrict__ part, int R, int C,
    const int64_t* __restrict__ state, uint32_t site, uint32_t threshold, float scale) {
  __shared__ float red[2][8][2 * kBwdRows];  // two buffers: one barrier per group of rows
  const int col = threadIdx.x * 8;
  const bool mine = col < C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const Draws draws(state, site);
  const uint32_t below = (threshold << 16) - 1;
  float aw[8], ab[8], ad[8], wf[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) aw[e] = ab[e] = ad[e] = wf[e] = 0.f;
  if (mine) unpack8(*reinterpret_cast<const uint4*>(w + col), wf);
  const uint4 z = make_uint4(0, 0, 0, 0);
  uint4 vg[kBwdRows], vs[kBwdRows], vr[kBwdRows];
  const int stride = gridDim.x * kBwdRows;
  int row0 = blockIdx.x * kBwdRows;
  auto load = [&](int r0) {
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) {
      const bool ok = mine && r0 + k < R;
      const size_t off = (size_t)(r0 + k) * C + col;
      vg[k] = ok ? stream16(dy + off) : z;
      vs[k] = ok ? stream16(s + off) : z;
      vr[k] = ok && dres ? stream16(dres + off) : z;
    }
  };
  load(row0);
  int buf = 0;
  for (; row0 < R; row0 += stride, buf ^= 1) {
    float mu[kBwdRows], rs[kBwdRows], sums[2 * kBwdRows];
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) {
      const bool ok = row0 + k < R;
      mu[k] = ok ? mean[row0 + k] : 0.f;
      rs[k] = ok ? rstd[row0 + k] : 0.f;
      float g[8], xh[8], s1 = 0.f, s2 = 0.f;
      unpack8(vg[k], g);
      unpack8(vs[k], xh);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[e] = (xh[e] - mu[k]) * rs[k];
        aw[e] += g[e] * xh[e];
        ab[e] += g[e];
        const float gw = g[e] * wf[e];
        s1 += gw;
        s2 += gw * xh[e];
      }
      sums[2 * k] = row_sum(s1);
      sums[2 * k + 1] = row_sum(s2);
    }
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < 2 * kBwdRows; ++k) red[buf][warp][k] = sums[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2 * kBwdRows; ++k) {
      float t = 0.f;
      for (int i = 0; i < warps; ++i) t += red[buf][i][k];
      sums[k] = t / C;
    }
    uint4 ox[kBwdRows], od[kBwdRows];
#pragma unroll
    for (int k = 0; k < kBwdRows; ++k) {
      float g[8], xh[8], o[8];
      unpack8(vg[k], g);
      unpack8(vs[k], xh);
      unpack8(vr[k], o);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[e] = (xh[e] - mu[k]) * rs[k];
        o[e] += rs[k] * (g[e] * wf[e] - sums[2 * k] - xh[e] * sums[2 * k + 1]);
      }
      ox[k] = pack8(o);
      drop8(o, draws(((size_t)(row0 + k) * C + col) >> 3), below, scale);
      od[k] = pack8(o);
      if constexpr (BIAS) {
        const bool ok = row0 + k < R;
#pragma unroll
        for (int e = 0; e < 8; ++e) ad[e] += ok ? o[e] : 0.f;  // before the rounding of dr
      }
    }
    const int done = row0;
    load(row0 + stride);
    if (mine) {
#pragma unroll
      for (int k = 0; k < kBwdRows; ++k) {
        if (done + k < R) {
          const size_t off = (size_t)(done + k) * C + col;
          *reinterpret_cast<uint4*>(dx + off) = ox[k];
          *reinterpret_cast<uint4*>(dr + off) = od[k];
        }
      }
    }
  }
  if (mine) {
    float4* p = reinterpret_cast<float4*>(part + (size_t)blockIdx.x * (BIAS ? 3 : 2) * C + col);
    const int c4 = C / 4;
    p[0] = make_float4(aw[0], aw[1], aw[2], aw[3]);
    p[1] = make_float4(aw[4], aw[5], aw[6], aw[7]);
    p[c4] = make_float4(ab[0], ab[1], ab[2], ab[3]);
    p[c4 + 1] = make_float4(ab[4], ab[5], ab[6], ab[7]);
    if constexpr (BIAS) {
      p[2 * c4] = make_float4(ad[0], ad[1], ad[2], ad[3]);
      p[2 * c4 + 1] = make_float4(ad[4], ad[5], ad[6], ad[7]);
    }
  }
}

// Column sums of the P partial rows of W = (2 or 3) C values, in a fixed order:
// 8 lanes of 4 columns by 32 slices of the partial rows per block.
__global__ void __launch_bounds__(256) k_dropout_ln_columns(const float* __restrict__ part, int P, int W, int C,
                                                            __nv_bfloat16* dw, __nv_bfloat16* db,
                                                            __nv_bfloat16* drb) {
  __shared__ float4 red[32][8];
  const int cg = threadIdx.x & 7, sl = threadIdx.x >> 3;
  const int col = (blockIdx.x * 8 + cg) * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < W) {
#pragma unroll 8
    for (int p = sl; p < P; p += 32) {
      const float4 v = *reinterpret_cast<const float4*>(part + (size_t)p * W + col);
      a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
  }
  red[sl][cg] = a;
  __syncthreads();
  if (threadIdx.x < 32) {  // one thread per column
    const int c1 = blockIdx.x * 32 + threadIdx.x;
    if (c1 < W) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) t += reinterpret_cast<const float*>(red[j])[threadIdx.x];
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
  if (drb)
    k_dropout_ln_bwd<true><<<grid, threads, 0, s>>>(dy, s_in, mean, rstd, w, dres, dx, dr, scratch, R, C, state, site,
                                                    threshold, scale);
  else
    k_dropout_ln_bwd<false><<<grid, threads, 0, s>>>(dy, s_in, mean, rstd, w, dres, dx, dr, scratch, R, C, state,
                                                     site, threshold, scale);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int W = (drb ? 3 : 2) * C;
  k_dropout_ln_columns<<<(W + 31) / 32, 256, 0, s>>>(scratch, grid, W, C, dw, db, drb);
  return cudaGetLastError();
}

}  // namespace nexar
