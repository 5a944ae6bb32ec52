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
// registers and takes several heads of its token, which makes the table's share
// of the L1 traffic small. Measured: 65537 tokens of 32 query and 8 key heads of
// 128, 96 elements of each turned (1.34 GB): 219 us, 6.1 TB/s; packed rows of 8 x
// 1024 tokens, 24 of 36 heads of 64 turned (75 MB): 14.2 us.
#include "decoder_api.h"
#include "pack.cuh"

namespace nexar {

namespace {
constexpr int kRotThreads = 256;
constexpr int kRotUnroll = 2;  // heads whose loads are in flight together
constexpr int kRotHeads = 4;   // heads per thread where there are many tokens

NEXAR_D long long rotary_position(const RotaryArgs& a, long long b, long long t) {
  if (!a.positions) return a.start + t;
  const long long at = b * a.pb + t * a.pt;
  return a.positions_64 ? reinterpret_cast<const long long*>(a.positions)[at]
                        : (long long)reinterpret_cast<const int*>(a.positions)[at];
}

// cos, sin of N pairs from `pair` on at a position; a position without a table row shows as NaN.
template <int N>
NEXAR_D void load_turn(const RotaryArgs& a, long long pos, int pair, float* c, float* s) {
  if (pos >= 0 && pos < a.rows) {
    const float* row = a.table + pos * a.R + 2 * pair;
    if constexpr (N % 2 == 0) {
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float4 v = *reinterpret_cast<const float4*>(row + 2 * e);
        c[e] = v.x, s[e] = a.sign * v.y, c[e + 1] = v.z, s[e + 1] = a.sign * v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 v = *reinterpret_cast<const float2*>(row + 2 * e);
        c[e] = v.x, s[e] = a.sign * v.y;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) c[e] = s[e] = __int_as_float(0x7fc00000);
  }
}

// The turn, rounded the same way wherever it is written: an fp32 result does not depend on the tensor's address.
NEXAR_D float turn_1(float x1, float x2, float c, float s) { return fmaf(x1, c, -(x2 * s)); }
NEXAR_D float turn_2(float x1, float x2, float c, float s) { return fmaf(x2, c, x1 * s); }

// Thread index -> (token, lane), with 32-bit division where it fits.
NEXAR_D void split_index(long long idx, long long threads, int lanes, long long* n, int* lane) {
  if (threads <= 0xffffffffLL) {
    *n = (unsigned)idx / (unsigned)lanes;
    *lane = (unsigned)idx % (unsigned)lanes;
  } else {
    *n = idx / lanes;
    *lane = (int)(idx % lanes);
  }
}

// A head is D / (2 W) slots of two packs of W elements. Half layout: a slot of
// the rotated part is a pack of first halves and the pack of their second
// halves; interleaved: packs i and i + D / (2 W). Slots behind the rotated part,
// and all slots of heads behind the rotated heads, are copied on the same path,
// so every thread has the loads of two heads (4 x 16 bytes) in flight whatever it
// does with them, and neighbouring threads touch neighbouring packs.
// A block works on one of the parts. One thread: token n, slot i, heads hg, hg + HG, ...
template <typename T, int W, bool INTER>
__global__ void __launch_bounds__(kRotThreads, 4) k_rotary(const __grid_constant__ RotaryArgs a, int slots,
                                                           unsigned blocks0, int HG0, int HG1, long long threads0,
                                                           long long threads1) {
  const bool second = blockIdx.x >= blocks0;
  const RotaryPart& p = a.part[second ? 1 : 0];
  const int HG = second ? HG1 : HG0;
  const long long threads = second ? threads1 : threads0;
  const long long idx = (blockIdx.x - (second ? blocks0 : 0u)) * (long long)kRotThreads + threadIdx.x;
  if (idx >= threads) return;
  long long n, b = 0, t;
  int lane, tt;
  split_index(idx, threads, slots * HG, &n, &lane);
  t = n;
  if (a.B > 1) {
    split_index(n, threads, (int)a.T, &b, &tt);
    t = tt;
  }
  const int hg = (unsigned)lane / (unsigned)slots, i = lane - hg * slots;
  // pack offsets of the slot, and which of its packs turn
  int o1, o2;
  bool turn1, turn2;
  float c[W], s[W];
  const long long pos = rotary_position(a, b, t);
  if constexpr (INTER) {
    o1 = i * W, o2 = a.D / 2 + i * W;
    turn1 = o1 < a.R, turn2 = o2 < a.R;
    if (turn1) load_turn<W / 2>(a, pos, o1 / 2, c, s);
    if (turn2) load_turn<W / 2>(a, pos, o2 / 2, c + W / 2, s + W / 2);
  } else {
    const int packs = a.R / (2 * W);
    turn1 = turn2 = i < packs;
    o1 = turn1 ? i * W : a.R + (i - packs) * W;
    o2 = o1 + (turn1 ? a.R : a.D - a.R) / 2;
    if (turn1) load_turn<W>(a, pos, i * W, c, s);
  }
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.sb + t * p.st + hg * p.sh;
  T* y = reinterpret_cast<T*>(p.y) + (n * p.heads + hg) * a.D;
  const long long dx = HG * p.sh;
  const long long dy = (long long)HG * a.D;
#pragma unroll 1
  for (int h0 = hg; h0 < p.heads; h0 += kRotUnroll * HG) {
    Pack<T, W> u[kRotUnroll], v[kRotUnroll];
#pragma unroll
    for (int k = 0; k < kRotUnroll; ++k) {
      if (h0 + k * HG < p.heads) u[k].load(x + k * dx + o1), v[k].load(x + k * dx + o2);
    }
#pragma unroll
    for (int k = 0; k < kRotUnroll; ++k) {
      const int h = h0 + k * HG;
      if (h < p.heads) {
        if constexpr (INTER) {
#pragma unroll
          for (int e = 0; e < W / 2; ++e) {
            if (turn1 && h < p.rotated) {
              const float2 z = u[k].get(e);
              u[k].set(e, turn_1(z.x, z.y, c[e], s[e]), turn_2(z.x, z.y, c[e], s[e]));
            }
            if (turn2 && h < p.rotated) {
              const float2 z = v[k].get(e);
              const float cc = c[W / 2 + e], ss = s[W / 2 + e];
              v[k].set(e, turn_1(z.x, z.y, cc, ss), turn_2(z.x, z.y, cc, ss));
            }
          }
        } else if (turn1 && h < p.rotated) {
#pragma unroll
          for (int e = 0; e < W / 2; ++e) {
            const float2 z1 = u[k].get(e), z2 = v[k].get(e);
            const float c0 = c[2 * e], s0 = s[2 * e], c1 = c[2 * e + 1], s1 = s[2 * e + 1];
            u[k].set(e, turn_1(z1.x, z2.x, c0, s0), turn_1(z1.y, z2.y, c1, s1));
            v[k].set(e, turn_2(z1.x, z2.x, c0, s0), turn_2(z1.y, z2.y, c1, s1));
          }
        }
        u[k].store(y + k * dy + o1);
        v[k].store(y + k * dy + o2);
      }
    }
    x += kRotUnroll * dx;
    y += kRotUnroll * dy;
  }
}

// Any sizes, strides and alignment: one pair per thread and element-wise
// accesses; what does not turn is copied element by element.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kRotThreads) k_rotary_any(const RotaryArgs a, int HG, long long threads) {
  const long long idx = blockIdx.x * (long long)kRotThreads + threadIdx.x;
  if (idx >= threads) return;
  const int pairs = a.R / 2;
  long long n;
  int lane;
  split_index(idx, threads, pairs * HG, &n, &lane);
  const int hg = lane / pairs, i = lane % pairs;
  const long long b = a.B == 1 ? 0 : n / a.T, t = n - b * a.T;
  float c, s;
  load_turn<1>(a, rotary_position(a, b, t), i, &c, &s);
  const int o1 = INTER ? 2 * i : i, o2 = INTER ? 2 * i + 1 : pairs + i;
  for (int part = 0; part < a.nparts; ++part) {
    const RotaryPart& p = a.part[part];
    for (int h = hg; h < p.heads; h += HG) {
      const T* x = reinterpret_cast<const T*>(p.x) + b * p.sb + t * p.st + h * p.sh;
      T* y = reinterpret_cast<T*>(p.y) + (n * p.heads + h) * a.D;
      if (h < p.rotated) {
        const float x1 = to_acc<float>(x[o1]), x2 = to_acc<float>(x[o2]);
        y[o1] = from_acc<T, float>(turn_1(x1, x2, c, s));
        y[o2] = from_acc<T, float>(turn_2(x1, x2, c, s));
      } else {
        y[o1] = x[o1], y[o2] = x[o2];
      }
      for (int j = a.R + i; j < a.D; j += pairs) y[j] = x[j];
    }
  }
}

// Few tokens: a thread per head, for the shortest path. Many: each thread takes
// kRotHeads heads of its token, so it reads the table once for them.
int head_groups(const RotaryArgs& a, int heads, int per_head) {
  return a.B * a.T * per_head * heads > 148LL * 2048 ? (heads + kRotHeads - 1) / kRotHeads : heads;
}

template <typename T, int W>
cudaError_t launch_rotary(const RotaryArgs& a, cudaStream_t s) {
  const int slots = a.D / (2 * W);
  int HG[2] = {1, 1};
  long long threads[2] = {0, 0}, blocks[2] = {0, 0};
  for (int p = 0; p < a.nparts; ++p) {
    HG[p] = head_groups(a, a.part[p].heads, slots);
    threads[p] = a.B * a.T * slots * HG[p];
    blocks[p] = (threads[p] + kRotThreads - 1) / kRotThreads;
  }
  if (blocks[0] + blocks[1] > 0x7fffffffLL || a.T > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)(blocks[0] + blocks[1]);
  if (a.interleaved)
    k_rotary<T, W, true><<<grid, kRotThreads, 0, s>>>(a, slots, (unsigned)blocks[0], HG[0], HG[1], threads[0], threads[1]);
  else
    k_rotary<T, W, false><<<grid, kRotThreads, 0, s>>>(a, slots, (unsigned)blocks[0], HG[0], HG[1], threads[0], threads[1]);
  return cudaGetLastError();
}
template <typename T> cudaError_t launch_rotary_any(const RotaryArgs& a, cudaStream_t s) {
  int heads = a.part[0].heads;
  if (a.nparts > 1 && a.part[1].heads > heads) heads = a.part[1].heads;
  const int pairs = a.R / 2, HG = head_groups(a, heads, pairs);
  const long long threads = a.B * a.T * pairs * HG, blocks = (threads + kRotThreads - 1) / kRotThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (a.interleaved)
    k_rotary_any<T, true><<<(unsigned)blocks, kRotThreads, 0, s>>>(a, HG, threads);
  else
    k_rotary_any<T, false><<<(unsigned)blocks, kRotThreads, 0, s>>>(a, HG, threads);
  return cudaGetLastError();
}

// The widest pack (elements) that sizes, strides and addresses allow, or 1.
int rotary_width(const RotaryArgs& a, int elem) {
  for (int w = 16 / elem; w >= 2; w /= 2) {
    bool ok = a.R % (a.interleaved ? w : 2 * w) == 0 && a.D % (2 * w) == 0;
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
    if (w == 8) return launch_rotary<T, 8>(a, s);
  }
  if (w == 4) return launch_rotary<T, 4>(a, s);
  if (w == 2) return launch_rotary<T, 2>(a, s);
  return launch_rotary_any<T>(a, s);
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
