// Rotary positions (sm_100a): every pair (x1, x2) of the first R elements of a
// head turns by the angle of its position,
//     y1 = x1 cos - x2 sin,   y2 = x2 cos + x1 sin,
// pairs (i, i + R/2) in the half layout and (2i, 2i + 1) in the interleaved
// one; the rest of the head is copied. The gradient is the same turn the other
// way (sign = -1).
//
// Bound by bandwidth: 2 bytes in and 2 out per element. The cosines and sines
// come from a table of fp32 pairs (built once in 64 bits by k_rotary_table, so
// far positions keep their angle); a thread keeps those of its pairs in
// registers and walks over several heads of its token, which makes the
// table's share of the L1 traffic small.
#include "common.cuh"
#include "decoder_api.h"

namespace nexar {

namespace {
constexpr int kRotThreads = 256;
constexpr int kRotUnroll = 4;  // heads whose loads are in flight together

// W elements of T as one load (VEC), or one by one where the alignment allows no wider one.
template <typename T, int W, bool VEC> struct Pack {
  T e[W];
};
template <typename T, int W> struct alignas(W * sizeof(T)) Pack<T, W, true> {
  T e[W];
};
template <typename T, int W, bool VEC> NEXAR_D Pack<T, W, VEC> load_pack(const T* p) {
  Pack<T, W, VEC> r;
  if constexpr (VEC && W * sizeof(T) == 16) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    memcpy(&r, &v, 16);
  } else if constexpr (VEC) {
    r = *reinterpret_cast<const Pack<T, W, true>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) r.e[i] = p[i];
  }
  return r;
}
template <typename T, int W, bool VEC> NEXAR_D void store_pack(T* p, const Pack<T, W, VEC>& r) {
  if constexpr (VEC) {
    *reinterpret_cast<Pack<T, W, true>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) p[i] = r.e[i];
  }
}

NEXAR_D long long rotary_position(const RotaryArgs& a, long long b, long long t) {
  if (!a.positions) return a.start + t;
  const long long at = b * a.pb + t * a.pt;
  return a.positions_64 ? reinterpret_cast<const long long*>(a.positions)[at]
                        : (long long)reinterpret_cast<const int*>(a.positions)[at];
}

// One thread: token n, pairs of pack i, heads hg, hg + HG, ...
// W: elements per pack; a pack holds W pairs' first halves (half layout, the
// second halves R/2 further) or W/2 whole pairs (interleaved).
template <typename T, int W, bool VEC, bool INTER>
__global__ void __launch_bounds__(kRotThreads) k_rotary(const RotaryArgs a, int packs, int HG, long long threads) {
  const long long idx = blockIdx.x * (long long)kRotThreads + threadIdx.x;
  if (idx >= threads) return;
  const int lanes = packs * HG;
  long long n;
  int lane;
  if (threads <= 0xffffffffLL) {  // 32-bit division where it fits
    n = (unsigned)idx / (unsigned)lanes;
    lane = (unsigned)idx % (unsigned)lanes;
  } else {
    n = idx / lanes;
    lane = (int)(idx % lanes);
  }
  const int hg = lane / packs, i = lane % packs;
  const long long b = a.B == 1 ? 0 : n / a.T, t = n - b * a.T;
  constexpr int NP = INTER ? W / 2 : W;  // pairs of a pack
  float c[NP], s[NP];
  const long long pos = rotary_position(a, b, t);
  if (pos >= 0 && pos < a.rows) {
    const float* row = a.table + pos * a.R + 2 * i * NP;
    if constexpr (NP % 2 == 0) {
#pragma unroll
      for (int e = 0; e < NP; e += 2) {
        const float4 v = *reinterpret_cast<const float4*>(row + 2 * e);
        c[e] = v.x, s[e] = a.sign * v.y, c[e + 1] = v.z, s[e + 1] = a.sign * v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        const float2 v = *reinterpret_cast<const float2*>(row + 2 * e);
        c[e] = v.x, s[e] = a.sign * v.y;
      }
    }
  } else {  // a position without a table row shows as NaN
#pragma unroll
    for (int e = 0; e < NP; ++e) c[e] = s[e] = __int_as_float(0x7fc00000);
  }
  const int half = a.R / 2;
  const int o1 = i * W, o2 = half + i * W;
  constexpr int CW = VEC ? W : 1;  // elements per copied pack: an odd head size has no pairs to copy
  const int tail = (a.D - a.R) / CW, whole = a.D / CW;
  using P = Pack<T, W, VEC>;
#pragma unroll 1
  for (int part = 0; part < a.nparts; ++part) {
    const RotaryPart& p = a.part[part];
    const T* x = reinterpret_cast<const T*>(p.x) + b * p.sb + t * p.st;
    T* y = reinterpret_cast<T*>(p.y) + n * p.heads * a.D;
#pragma unroll 1
    for (int h0 = hg; h0 < p.rotated; h0 += kRotUnroll * HG) {
      P u[kRotUnroll], v[INTER ? 1 : kRotUnroll];
#pragma unroll
      for (int k = 0; k < kRotUnroll; ++k) {
        const int h = h0 + k * HG;
        if (h < p.rotated) {
          const T* q = x + h * p.sh;
          u[k] = load_pack<T, W, VEC>(q + o1);
          if constexpr (!INTER) v[k] = load_pack<T, W, VEC>(q + o2);
        }
      }
#pragma unroll
      for (int k = 0; k < kRotUnroll; ++k) {
        const int h = h0 + k * HG;
        if (h < p.rotated) {
          T* q = y + (long long)h * a.D;
          if constexpr (INTER) {
#pragma unroll
            for (int e = 0; e < NP; ++e) {
              const float x1 = to_acc<float>(u[k].e[2 * e]), x2 = to_acc<float>(u[k].e[2 * e + 1]);
              u[k].e[2 * e] = from_acc<T, float>(x1 * c[e] - x2 * s[e]);
              u[k].e[2 * e + 1] = from_acc<T, float>(x2 * c[e] + x1 * s[e]);
            }
            store_pack<T, W, VEC>(q + o1, u[k]);
          } else {
#pragma unroll
            for (int e = 0; e < NP; ++e) {
              const float x1 = to_acc<float>(u[k].e[e]), x2 = to_acc<float>(v[k].e[e]);
              u[k].e[e] = from_acc<T, float>(x1 * c[e] - x2 * s[e]);
              v[k].e[e] = from_acc<T, float>(x2 * c[e] + x1 * s[e]);
            }
            store_pack<T, W, VEC>(q + o1, u[k]);
            store_pack<T, W, VEC>(q + o2, v[k]);
          }
        }
      }
    }
    // what is not rotated: the heads' tails, and whole heads behind the rotated ones
    if (tail) {
#pragma unroll 1
      for (int h = hg; h < p.rotated; h += HG)
#pragma unroll 1
        for (int j = i; j < tail; j += packs)
          store_pack<T, CW, VEC>(y + (long long)h * a.D + a.R + j * CW,
                                 load_pack<T, CW, VEC>(x + h * p.sh + a.R + j * CW));
    }
#pragma unroll 1
    for (int h = p.rotated + hg; h < p.heads; h += HG)
#pragma unroll 2
      for (int j = i; j < whole; j += packs)
        store_pack<T, CW, VEC>(y + (long long)h * a.D + j * CW, load_pack<T, CW, VEC>(x + h * p.sh + j * CW));
  }
}

template <typename T, int W, bool VEC>
cudaError_t launch_rotary(const RotaryArgs& a, cudaStream_t s) {
  const int packs = a.interleaved ? a.R / W : a.R / (2 * W);
  int heads = 1;
  for (int p = 0; p < a.nparts; ++p) heads = a.part[p].heads > heads ? a.part[p].heads : heads;
  // Few tokens: a thread per head, for the shortest path. Many: each thread
  // takes four heads of its token, so it reads the table once for them.
  const long long tokens = a.B * a.T;
  int HG = heads;
  if (tokens * packs * heads > 148LL * 2048) HG = (heads + kRotUnroll - 1) / kRotUnroll;
  const long long threads = tokens * packs * HG;
  const long long blocks = (threads + kRotThreads - 1) / kRotThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (a.interleaved) {
    if constexpr (W >= 2)
      k_rotary<T, W, VEC, true><<<(unsigned)blocks, kRotThreads, 0, s>>>(a, packs, HG, threads);
    else
      return cudaErrorInvalidValue;
  } else {
    k_rotary<T, W, VEC, false><<<(unsigned)blocks, kRotThreads, 0, s>>>(a, packs, HG, threads);
  }
  return cudaGetLastError();
}

// The widest pack that sizes, strides and addresses allow.
int rotary_width(const RotaryArgs& a, int elem) {
  for (int w = 16 / elem; w >= 2; w /= 2) {
    const int per = a.interleaved ? w : 2 * w;
    bool ok = a.R % per == 0 && a.D % w == 0;
    for (int p = 0; ok && p < a.nparts; ++p) {
      const RotaryPart& q = a.part[p];
      ok = q.sb % w == 0 && q.st % w == 0 && q.sh % w == 0 && (uintptr_t)q.x % (w * elem) == 0 &&
           (uintptr_t)q.y % (w * elem) == 0;
    }
    if (ok) return w;
  }
  return 1;
}

__global__ void __launch_bounds__(256) k_rotary_table(const double* __restrict__ freq, float2* __restrict__ table,
                                                      long long n, int half, double magnitude) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= n) return;
  double sn, cs;
  sincos((double)(i / half) * freq[i % half], &sn, &cs);
  table[i] = make_float2((float)(magnitude * cs), (float)(magnitude * sn));
}
}  // namespace

template <typename T> static cudaError_t rotary_typed(const RotaryArgs& a, cudaStream_t s) {
  const int w = rotary_width(a, sizeof(T));
  if constexpr (sizeof(T) == 2) {
    if (w == 8) return launch_rotary<T, 8, true>(a, s);
  }
  if (w == 4) return launch_rotary<T, 4, true>(a, s);
  if (w == 2) return launch_rotary<T, 2, true>(a, s);
  // interleaved pairs stay together: two elements, read one by one
  return a.interleaved ? launch_rotary<T, 2, false>(a, s) : launch_rotary<T, 1, false>(a, s);
}

cudaError_t rotary(const RotaryArgs& a, int elem, bool half, cudaStream_t s) {
  if (a.R <= 0 || a.R % 2 || a.R > a.D || a.nparts < 1 || a.nparts > 2) return cudaErrorInvalidValue;
  if (a.B * a.T == 0) return cudaSuccess;
  if (elem == 4) return rotary_typed<float>(a, s);
  return half ? rotary_typed<__half>(a, s) : rotary_typed<__nv_bfloat16>(a, s);
}

cudaError_t rotary_table(const double* freq, float* table, long long rows, int R, double magnitude, cudaStream_t s) {
  const long long n = rows * (R / 2);
  if (n <= 0 || (n + 255) / 256 > 0x7fffffffLL) return cudaErrorInvalidValue;
  k_rotary_table<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(freq, reinterpret_cast<float2*>(table), n, R / 2,
                                                             magnitude);
  return cudaGetLastError();
}

}  // namespace nexar
