// Norm of every query and key head and the rotation by the token's position, in one pass, forward and backward (gfx950).
//
//   z = x r w,  r = 1 / sqrt(mean(x^2) + eps);   pair (a, b) of z -> (a cos t - b sin t, a sin t + b cos t),  t = position[axis(pair)] inv_freq[pair]
//   dz = rotation by -t of dy;  dw = sum over tokens and heads of dz x r;  dx = r w dz - x r^3 mean(w dz x)
//
// Bound by memory: each head is read once and written once (backward: x and dy read, dx written): 30000 tokens x 20 heads of 128 (bf16) take
// 73 us forward = 4.2 TB/s and 119 us backward = 3.9 TB/s, where a large copy reaches 4.6.  A row (one head of one token) belongs to
// dim / (2 V) neighbouring lanes; a lane holds V channels and their V partners, so a rotation stays inside a lane, and the sums over a head
// are a few exchanges between neighbours.  The angles belong to the token: a lane computes its sines and cosines once and keeps them for
// all heads of its token.
//
// Angles.  pos * inv_freq is formed in revolutions in 64 bits (three roundings: off by 2^-51 of itself at most) and reduced to half a turn there: at
// position 10^6 a 32-bit product is off by 0.06 rad, this one by 4 10^-10.  16-bit heads: the rest is rounded to 32 bits and goes to the hardware's sine and
// cosine, which take turns: off by 2.2 10^-7 with the rounding, a 2000th of fp16's half step.  32-bit heads, where that would be three half steps: Taylor's
// series in 64 bits on an eighth of a turn, rounded once (once for all heads of a token: 10.5 -> 11.1 us at 9000 tokens x 12 heads of 40).
#include "common.h"
#include <algorithm>
#include <string.h>

namespace {
using namespace dh;

struct IoF32 {
  static constexpr int SIZE = 4, VMAX = 4;
  static __device__ __forceinline__ float get(const char* p, int i) { return reinterpret_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ void put(char* p, int i, float v) { reinterpret_cast<float*>(p)[i] = v; }
};
struct IoF16 {
  static constexpr int SIZE = 2, VMAX = 8;
  static __device__ __forceinline__ float get(const char* p, int i) { return (float)reinterpret_cast<const _Float16*>(p)[i]; }
  static __device__ __forceinline__ void put(char* p, int i, float v) { reinterpret_cast<_Float16*>(p)[i] = (_Float16)v; }
};
struct IoBF16 {
  static constexpr int SIZE = 2, VMAX = 8;
  static __device__ __forceinline__ float get(const char* p, int i) { return (float)reinterpret_cast<const __bf16*>(p)[i]; }
  static __device__ __forceinline__ void put(char* p, int i, float v) { reinterpret_cast<__bf16*>(p)[i] = (__bf16)v; }
};

// V values with one load / store of V * SIZE bytes
template <int BYTES> struct Raw { typedef unsigned char type; };
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef unsigned type; };
template <> struct Raw<2> { typedef unsigned short type; };
template <typename Io, int V> struct Vec {
  typename Raw<V * Io::SIZE>::type raw;
  __device__ __forceinline__ void load(const char* p) { raw = *reinterpret_cast<const decltype(raw)*>(p); }
  __device__ __forceinline__ void store(char* p) const { *reinterpret_cast<decltype(raw)*>(p) = raw; }
  __device__ __forceinline__ float get(int i) const { return Io::get(reinterpret_cast<const char*>(&raw), i); }
  __device__ __forceinline__ void put(int i, float v) { Io::put(reinterpret_cast<char*>(&raw), i, v); }
};

struct Tensor { char* p; long st, sh; };          // base, bytes between tokens, bytes between heads

struct RopeParams {
  Tensor x[2], y[2], g[2];                       // q and k; forward: y = result; backward: g = gradient of the result, y = gradient of x
  int heads[2];
  const void* w[2];
  int w_type, pos_type, n_axes, sect_end[4];
  const void* pos;
  const float* inv_freq;
  float* part;                                   // backward: [workgroups][2][dim] partial sums of dw
  long tokens;
  int dim, pairs, shift, chunk;                  // shift: log2 of the lanes a row has; chunk: heads a workgroup takes (grid.y)
  float eps, inv_dim;
};

__device__ __forceinline__ float weight_at(const void* w, int type, int i) {
  if (!w) return 1.f;
  return type == DH_F32 ? reinterpret_cast<const float*>(w)[i] : type == DH_F16 ? (float)reinterpret_cast<const _Float16*>(w)[i] : (float)reinterpret_cast<const __bf16*>(w)[i];
}

// What a lane knows about its chunk of a row: where its V channels and their V partners lie.
template <int V, bool PAIRS_ADJACENT> struct Lane {
  int lo, hi;                                    // first channels
  bool on;
  __device__ __forceinline__ Lane(const RopeParams& p, int c) {
    on = c < p.dim / (2 * V);
    if (!on) c = 0;
    if (PAIRS_ADJACENT) { lo = 2 * c * V; hi = lo + V; }
    else if (c * V < p.pairs) { lo = c * V; hi = p.pairs + lo; }
    else { lo = p.pairs + c * V; hi = lo + p.dim / 2 - p.pairs; }            // channels that do not turn
  }
  // first pair of the chunk (>= pairs: it does not turn)
  __device__ __forceinline__ int pair(int i) const { return PAIRS_ADJACENT ? lo / 2 + i : lo + i; }
};

// sin and cos of `rev` turns, |rev| <= 1/2, rounded to 32 bits once: the nearest quarter turn is taken off, and the series to x^13 and x^12 are off by
// 4 10^-13 where |x| <= pi / 4
__device__ __forceinline__ void sincos_turns(double rev, float& s, float& c) {
  const int n = (int)rint(4. * rev);
  const double x = (rev - .25 * n) * 6.28318530717958647693, y = x * x;
  const double si = x + x * y * (-1. / 6 + y * (1. / 120 + y * (-1. / 5040 + y * (1. / 362880 + y * (-1. / 39916800 + y * (1. / 6227020800.))))));
  const double co = 1. + y * (-1. / 2 + y * (1. / 24 + y * (-1. / 720 + y * (1. / 40320 + y * (-1. / 3628800 + y * (1. / 479001600.))))));
  const float a = (float)(n & 1 ? co : si), b = (float)(n & 1 ? si : co);
  s = n & 2 ? -a : a;
  c = (n + 1) & 2 ? -b : b;
}

template <int V> struct Turn { float c[V], s[V]; };
template <typename Io, int V, bool ADJ> __device__ __forceinline__ Turn<V> turn_of(const RopeParams& p, const Lane<V, ADJ>& ln, long tok) {
  Turn<V> t;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int j = ln.pair(i);
    t.c[i] = 1.f;
    t.s[i] = 0.f;
    if (j < p.pairs) {
      int axis = 0;
#pragma unroll
      for (int a = 0; a < 3; ++a) axis += a + 1 < p.n_axes && j >= p.sect_end[a];
      const long at = tok * p.n_axes + axis;
      const double x = p.pos_type == 0 ? (double)reinterpret_cast<const int*>(p.pos)[at]
                     : p.pos_type == 1 ? (double)reinterpret_cast<const long*>(p.pos)[at] : (double)reinterpret_cast<const float*>(p.pos)[at];
      const double rev = x * ((double)p.inv_freq[j] * 0.15915494309189533577);
      if constexpr (Io::SIZE == 4) {
        sincos_turns(rev - rint(rev), t.s[i], t.c[i]);
        continue;
      }
      const float turn = (float)(rev - rint(rev));                           // half a turn at most
      t.s[i] = __builtin_amdgcn_sinf(turn);                                  // v_sin_f32, v_cos_f32: argument in turns, off by 1.25e-7 at most
      t.c[i] = __builtin_amdgcn_cosf(turn);                                  // on [-1/2, 1/2] (all 2^22 multiples of 2^-22 compared with 64 bits)
    }
  }
  return t;
}
// rotates the chunk's pairs: a = first V channels, b = second V; adjacent pairs are (a0, a1), (a2, a3) .. (b0, b1) ..
template <int V, bool ADJ> __device__ __forceinline__ void rotate(float* a, float* b, const Turn<V>& t, float sign) {
  if constexpr (ADJ && V == 1) {
    const float x = a[0], y = b[0], s = t.s[0] * sign;
    a[0] = x * t.c[0] - y * s;
    b[0] = x * s + y * t.c[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float& u = ADJ ? (i < V / 2 ? a[2 * i] : b[2 * i - V]) : a[i];
      float& v = ADJ ? (i < V / 2 ? a[2 * i + 1] : b[2 * i + 1 - V]) : b[i];
      const float x = u, y = v, s = t.s[i] * sign;
      u = x * t.c[i] - y * s;
      v = x * s + y * t.c[i];
    }
  }
}
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over the 2^shift lanes of a row, in every one of them: neighbours, pairs, quads (mirrored in 8 lanes), eights (mirrored in 16)
__device__ __forceinline__ float row_sum(float v, int shift) {
  if (shift > 0) v += dpp<0xB1>(v);
  if (shift > 1) v += dpp<0x4E>(v);
  if (shift > 2) v += dpp<0x141>(v);
  if (shift > 3) v += dpp<0x140>(v);
  if (shift > 4) v += __shfl_xor(v, 16, 64);
  if (shift > 5) v += __shfl_xor(v, 32, 64);
  return v;
}

constexpr int FWD_HEADS = 4, BWD_HEADS = 2;      // heads whose loads are in flight together

template <typename Io, int V, bool ADJ, bool NORM>
__global__ __launch_bounds__(256, 4) void rope_fwd_kernel(const RopeParams p) {
  const int lane = threadIdx.x & 63, slots = 64 >> p.shift;
  const long tok = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * slots + (lane >> p.shift);
  const Lane<V, ADJ> ln(p, lane & ((1 << p.shift) - 1));
  const bool on = ln.on && tok < p.tokens;
  const long tk = tok < p.tokens ? tok : p.tokens - 1;
  const Turn<V> t = turn_of<Io, V, ADJ>(p, ln, tk);
  const int h_from = blockIdx.y * p.chunk, h_to = h_from + p.chunk;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int base = n ? p.heads[0] : 0;
    const int h0 = max(h_from - base, 0), h1 = min(h_to - base, p.heads[n]);
    if (h0 >= h1) continue;
    float wa[V], wb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      wa[i] = NORM ? weight_at(p.w[n], p.w_type, ln.lo + i) : 1.f;
      wb[i] = NORM ? weight_at(p.w[n], p.w_type, ln.hi + i) : 1.f;
    }
    const char* xp = p.x[n].p + tk * p.x[n].st;
    char* yp = p.y[n].p + tk * p.y[n].st;
    for (int h = h0; h < h1; h += FWD_HEADS) {
      Vec<Io, V> xa[FWD_HEADS], xb[FWD_HEADS];
#pragma unroll
      for (int u = 0; u < FWD_HEADS; ++u) {                                  // (the last head stands in for those behind it)
        const long at = min(h + u, h1 - 1) * p.x[n].sh;
        xa[u].load(xp + at + ln.lo * Io::SIZE);
        xb[u].load(xp + at + ln.hi * Io::SIZE);
      }
#pragma unroll
      for (int u = 0; u < FWD_HEADS; ++u) {
        float a[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { a[i] = xa[u].get(i); b[i] = xb[u].get(i); }
        if (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) ss += a[i] * a[i] + b[i] * b[i];
          const float r = rsqrtf(row_sum(ln.on ? ss : 0.f, p.shift) * p.inv_dim + p.eps);
#pragma unroll
          for (int i = 0; i < V; ++i) { a[i] *= r * wa[i]; b[i] *= r * wb[i]; }
        }
        rotate<V, ADJ>(a, b, t, 1.f);
#pragma unroll
        for (int i = 0; i < V; ++i) { xa[u].put(i, a[i]); xb[u].put(i, b[i]); }
      }
#pragma unroll
      for (int u = 0; u < FWD_HEADS; ++u)
        if (on && h + u < h1) {
          char* to = yp + (h + u) * p.y[n].sh;
          xa[u].store(to + ln.lo * Io::SIZE);
          xb[u].store(to + ln.hi * Io::SIZE);
        }
    }
  }
}

// Workgroups walk over the tokens with a fixed stride, so that the sums of dw stay in registers; their order does not depend on timing.
template <typename Io, int V, bool ADJ, bool NORM>
__global__ __launch_bounds__(256) void rope_bwd_kernel(const RopeParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slots = 64 >> p.shift;
  const Lane<V, ADJ> ln(p, lane & ((1 << p.shift) - 1));
  const int h_from = blockIdx.y * p.chunk, h_to = h_from + p.chunk;
  float sum[2][2][V];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) sum[n][0][i] = sum[n][1][i] = 0.f;
  for (long t0 = (long)blockIdx.x * 4 * slots; t0 < p.tokens; t0 += (long)gridDim.x * 4 * slots) {
    const long tok = t0 + wave * slots + (lane >> p.shift);
    const bool on = ln.on && tok < p.tokens;
    const long tk = tok < p.tokens ? tok : p.tokens - 1;
    const Turn<V> t = turn_of<Io, V, ADJ>(p, ln, tk);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int base = n ? p.heads[0] : 0;
      const int h0 = max(h_from - base, 0), h1 = min(h_to - base, p.heads[n]);
      if (h0 >= h1) continue;
      float wa[V], wb[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        wa[i] = NORM ? weight_at(p.w[n], p.w_type, ln.lo + i) : 1.f;
        wb[i] = NORM ? weight_at(p.w[n], p.w_type, ln.hi + i) : 1.f;
      }
      const char* xp = p.x[n].p + tk * p.x[n].st;
      const char* gp = p.g[n].p + tk * p.g[n].st;
      char* yp = p.y[n].p + tk * p.y[n].st;
      for (int h = h0; h < h1; h += BWD_HEADS) {
        Vec<Io, V> ga[BWD_HEADS], gb[BWD_HEADS], va[BWD_HEADS], vb[BWD_HEADS];
#pragma unroll
        for (int u = 0; u < BWD_HEADS; ++u) {
          const long hh = min(h + u, h1 - 1);
          ga[u].load(gp + hh * p.g[n].sh + ln.lo * Io::SIZE);
          gb[u].load(gp + hh * p.g[n].sh + ln.hi * Io::SIZE);
          if (NORM) {
            va[u].load(xp + hh * p.x[n].sh + ln.lo * Io::SIZE);
            vb[u].load(xp + hh * p.x[n].sh + ln.hi * Io::SIZE);
          }
        }
#pragma unroll
        for (int u = 0; u < BWD_HEADS; ++u) {
          float a[V], b[V];
#pragma unroll
          for (int i = 0; i < V; ++i) { a[i] = ga[u].get(i); b[i] = gb[u].get(i); }
          rotate<V, ADJ>(a, b, t, -1.f);
          if (NORM) {
            float ss = 0.f, sx = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float xa = va[u].get(i), xb = vb[u].get(i);
              ss += xa * xa + xb * xb;
              sx += wa[i] * a[i] * xa + wb[i] * b[i] * xb;
            }
            const float r = rsqrtf(row_sum(ln.on ? ss : 0.f, p.shift) * p.inv_dim + p.eps);
            const float m = row_sum(ln.on ? sx : 0.f, p.shift) * p.inv_dim * r * r * r;
            const bool count = on && h + u < h1;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float xa = va[u].get(i), xb = vb[u].get(i);
              if (count) { sum[n][0][i] += a[i] * xa * r; sum[n][1][i] += b[i] * xb * r; }
              a[i] = r * wa[i] * a[i] - xa * m;
              b[i] = r * wb[i] * b[i] - xb * m;
            }
          }
#pragma unroll
          for (int i = 0; i < V; ++i) { ga[u].put(i, a[i]); gb[u].put(i, b[i]); }
        }
#pragma unroll
        for (int u = 0; u < BWD_HEADS; ++u)
          if (on && h + u < h1) {
            char* to = yp + (h + u) * p.y[n].sh;
            ga[u].store(to + ln.lo * Io::SIZE);
            gb[u].store(to + ln.hi * Io::SIZE);
          }
      }
    }
  }
  if (!NORM || !p.part) return;
  __shared__ float red[4][2][256];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = sum[n][u][i];
        for (int k = p.shift; k < 6; ++k) v += __shfl_xor(v, 1 << k, 64);
        if (ln.on && lane < (1 << p.shift)) red[wave][n][(u ? ln.hi : ln.lo) + i] = v;
      }
  __syncthreads();
  float* out = p.part + ((long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.dim;
  for (int i = threadIdx.x; i < 2 * p.dim; i += 256) {
    const int n = i >= p.dim, d = i - n * p.dim;
    out[i] = red[0][n][d] + red[1][n][d] + red[2][n][d] + red[3][n][d];
  }
}

// dw[n][d] = sum over the workgroups' partial sums; 8 columns a workgroup, 32 threads a column
__global__ __launch_bounds__(256) void rope_dw_kernel(const float* __restrict__ part, int blocks, int dim, void* dq, void* dk, int w_type) {
  __shared__ float red[32][9];
  const int col = blockIdx.x * 8 + (threadIdx.x & 7), grp = threadIdx.x >> 3;
  float s = 0.f;
  if (col < 2 * dim)
    for (int b = grp; b < blocks; b += 32) s += part[(long)b * 2 * dim + col];
  red[grp][threadIdx.x & 7] = s;
  __syncthreads();
  if (grp || col >= 2 * dim) return;
  float v = 0.f;
  for (int g = 0; g < 32; ++g) v += red[g][threadIdx.x];
  void* out = col < dim ? dq : dk;
  const int d = col < dim ? col : col - dim;
  if (!out) return;
  if (w_type == DH_F32) reinterpret_cast<float*>(out)[d] = v;
  else if (w_type == DH_F16) reinterpret_cast<_Float16*>(out)[d] = (_Float16)v;
  else reinterpret_cast<__bf16*>(out)[d] = (__bf16)v;
}

constexpr int BWD_BLOCKS = 512;                  // two workgroups a CU is what their registers allow: one round (1024: 146 instead of 130 us on 30000 tokens)

bool tensor_ok(const Tensor& t, long tokens, int heads, int size) {
  if (!tokens || !heads) return true;
  return t.p && t.st >= 0 && t.sh >= 0 && t.st < (1l << 40) && t.sh < (1l << 40) && t.st % size == 0 && t.sh % size == 0 && (unsigned long)t.p % size == 0;
}
bool aligned(const Tensor& t, int heads, long bytes) {
  return !heads || (((unsigned long)t.p | (unsigned long)t.st | (unsigned long)t.sh) % bytes == 0);
}

// how many neighbouring channels a lane can hold: they divide the turning and the resting half of a row, and their bytes every address
int vector_of(const RopeParams& p, bool adjacent, int size, bool bwd) {
  int v = 16 / size;
  for (; v > 1; v /= 2) {
    bool ok = (p.dim / 2) % v == 0 && (adjacent || p.pairs % v == 0);
    for (int n = 0; n < 2; ++n) ok = ok && aligned(p.x[n], p.heads[n], v * size) && aligned(p.y[n], p.heads[n], v * size) && (!bwd || aligned(p.g[n], p.heads[n], v * size));
    if (ok) break;
  }
  return v;
}

template <typename Io, int V, bool ADJ, bool NORM> int launch(RopeParams& p, bool bwd, int* blocks, hipStream_t st) {
  const int lanes = p.dim / (2 * V);
  if (lanes > 64) return DH_ERR_UNSUPPORTED;
  p.shift = 0;
  while ((1 << p.shift) < lanes) ++p.shift;
  const int slots = 64 >> p.shift, total = p.heads[0] + p.heads[1];
  const long groups = (p.tokens + 4 * slots - 1) / (4 * slots);
  // few tokens: the heads are spread over workgroups as well, until every place on the chip has one: four a CU forward, two backward (5376 tokens x
  // 16 heads of 64: forward 10.2 us, with two 11.0, with eight 14.4; backward 21 us, with four 32)
  const int parts = (int)std::min<long>(total, std::max<long>(1, (bwd ? 512 : 1024) / groups));
  p.chunk = (total + parts - 1) / parts;
  const int gy = (total + p.chunk - 1) / p.chunk;
  if (!bwd) {
    if (groups > 0xffffffffl / 256) return DH_ERR_ARG;                       // threads of one launch
    hipLaunchKernelGGL((rope_fwd_kernel<Io, V, ADJ, NORM>), dim3((unsigned)groups, gy), dim3(256), 0, st, p);
  } else {
    const int gx = (int)std::min<long>(groups, std::max(1, BWD_BLOCKS / gy));
    *blocks = gx * gy;
    hipLaunchKernelGGL((rope_bwd_kernel<Io, V, ADJ, NORM>), dim3(gx, gy), dim3(256), 0, st, p);
  }
  DH_LAUNCH_CHECK();
  return DH_OK;
}
template <typename Io, int V> int pick(RopeParams& p, bool adjacent, bool norm, bool bwd, int* blocks, hipStream_t st) {
  if constexpr (V <= Io::VMAX) {
    if (adjacent) return norm ? launch<Io, V, true, true>(p, bwd, blocks, st) : launch<Io, V, true, false>(p, bwd, blocks, st);
    return norm ? launch<Io, V, false, true>(p, bwd, blocks, st) : launch<Io, V, false, false>(p, bwd, blocks, st);
  }
  return DH_ERR_UNSUPPORTED;
}
template <typename Io> int pick_v(RopeParams& p, bool adjacent, bool norm, bool bwd, int* blocks, hipStream_t st) {
  // the backward holds x, dy and the sums of dw: with 8 channels and their partners a lane it needs over 256 registers, one wave a SIMD (30000
  // tokens x 20 heads of 128: 177 us against 134 with 4 channels)
  const int v = std::min(bwd ? 4 : 8, vector_of(p, adjacent, Io::SIZE, bwd));
  return v == 8 ? pick<Io, 8>(p, adjacent, norm, bwd, blocks, st) : v == 4 ? pick<Io, 4>(p, adjacent, norm, bwd, blocks, st)
       : v == 2 ? pick<Io, 2>(p, adjacent, norm, bwd, blocks, st) : pick<Io, 1>(p, adjacent, norm, bwd, blocks, st);
}

int fill(RopeParams& p, const void* positions, int pos_type, const float* inv_freq, const int* sections, int n_axes, const void* qw, const void* kw, int w_type, int dtype,
         int64_t tokens, int heads, int kv_heads, int dim, int normalize, float eps) {
  if ((dtype != DH_F16 && dtype != DH_BF16 && dtype != DH_F32) || (w_type != DH_F16 && w_type != DH_BF16 && w_type != DH_F32) || pos_type < 0 || pos_type > 2 || tokens < 0 ||
      tokens > (1l << 40) || heads < 0 || kv_heads < 0 || heads > 4096 || kv_heads > 4096 || dim < 2 || dim > 256 || dim % 2 || n_axes < 1 || n_axes > 4 || !sections ||
      !(eps >= 0.f)) return DH_ERR_ARG;
  if (!normalize && (qw || kw)) return DH_ERR_ARG;
  int at = 0;
  for (int a = 0; a < 4; ++a) {
    if (a < n_axes) {
      if (sections[a] < 0 || sections[a] > dim) return DH_ERR_ARG;
      at += sections[a];
    }
    p.sect_end[a] = at;
  }
  if (at > dim / 2) return DH_ERR_ARG;
  if (tokens && heads + kv_heads && at && (!positions || !inv_freq)) return DH_ERR_ARG;
  p.pairs = at;
  p.heads[0] = heads; p.heads[1] = kv_heads;
  p.w[0] = qw; p.w[1] = kw; p.w_type = w_type;
  p.pos_type = pos_type; p.n_axes = n_axes; p.pos = positions; p.inv_freq = inv_freq;
  p.tokens = tokens; p.dim = dim; p.eps = eps; p.inv_dim = 1.f / (float)dim;
  return DH_OK;
}
Tensor tensor(const void* p, int64_t st, int64_t sh, int size) { return Tensor{(char*)const_cast<void*>(p), (long)st * size, (long)sh * size}; }

int run(RopeParams& p, int dtype, int interleaved, int normalize, bool bwd, int* blocks, hipStream_t st) {
  const bool adj = interleaved != 0, norm = normalize != 0;
  if (dtype == DH_F32) return pick_v<IoF32>(p, adj, norm, bwd, blocks, st);
  if (dtype == DH_F16) return pick_v<IoF16>(p, adj, norm, bwd, blocks, st);
  return pick_v<IoBF16>(p, adj, norm, bwd, blocks, st);
}

}  // namespace

extern "C" int dh_qk_norm_rope_fwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, void* q_out, int64_t qo_st, int64_t qo_sh,
                                   void* k_out, int64_t ko_st, int64_t ko_sh, const void* positions, int pos_type, const float* inv_freq, const int* sections_host,
                                   int n_axes, const void* q_weight, const void* k_weight, int w_dtype, int dtype, int64_t tokens, int heads, int kv_heads, int head_dim,
                                   int normalize, float eps, int interleaved, dh_stream_t stream) {
  RopeParams p;
  memset(&p, 0, sizeof p);
  const int rc = fill(p, positions, pos_type, inv_freq, sections_host, n_axes, q_weight, k_weight, w_dtype, dtype, tokens, heads, kv_heads, head_dim, normalize, eps);
  if (rc != DH_OK) return rc;
  if (tokens == 0 || heads + kv_heads == 0) return DH_OK;
  const int size = dtype == DH_F32 ? 4 : 2;
  p.x[0] = tensor(q, q_st, q_sh, size); p.x[1] = tensor(k, k_st, k_sh, size);
  p.y[0] = tensor(q_out, qo_st, qo_sh, size); p.y[1] = tensor(k_out, ko_st, ko_sh, size);
  for (int n = 0; n < 2; ++n)
    if (!tensor_ok(p.x[n], tokens, p.heads[n], size) || !tensor_ok(p.y[n], tokens, p.heads[n], size)) return DH_ERR_ARG;
  return run(p, dtype, interleaved, normalize, false, nullptr, (hipStream_t)stream);
}

extern "C" size_t dh_qk_norm_rope_bwd_workspace_bytes(int head_dim) {
  return head_dim >= 2 && head_dim <= 256 ? (size_t)BWD_BLOCKS * 2 * head_dim * sizeof(float) : 0;
}

extern "C" int dh_qk_norm_rope_bwd(const void* dq_out, int64_t gq_st, int64_t gq_sh, const void* dk_out, int64_t gk_st, int64_t gk_sh, const void* q, int64_t q_st, int64_t q_sh,
                                   const void* k, int64_t k_st, int64_t k_sh, void* dq, int64_t dq_st, int64_t dq_sh, void* dk, int64_t dk_st, int64_t dk_sh,
                                   void* dq_weight, void* dk_weight, const void* positions, int pos_type, const float* inv_freq, const int* sections_host, int n_axes,
                                   const void* q_weight, const void* k_weight, int w_dtype, int dtype, int64_t tokens, int heads, int kv_heads, int head_dim, int normalize,
                                   float eps, int interleaved, void* workspace, size_t workspace_bytes, dh_stream_t stream) {
  RopeParams p;
  memset(&p, 0, sizeof p);
  const int rc = fill(p, positions, pos_type, inv_freq, sections_host, n_axes, q_weight, k_weight, w_dtype, dtype, tokens, heads, kv_heads, head_dim, normalize, eps);
  if (rc != DH_OK) return rc;
  if (!normalize && (dq_weight || dk_weight)) return DH_ERR_ARG;
  const bool want_w = dq_weight || dk_weight;
  if (want_w && (!workspace || workspace_bytes < dh_qk_norm_rope_bwd_workspace_bytes(head_dim))) return DH_ERR_WORKSPACE;
  const int size = dtype == DH_F32 ? 4 : 2;
  p.x[0] = tensor(q, q_st, q_sh, size); p.x[1] = tensor(k, k_st, k_sh, size);
  p.g[0] = tensor(dq_out, gq_st, gq_sh, size); p.g[1] = tensor(dk_out, gk_st, gk_sh, size);
  p.y[0] = tensor(dq, dq_st, dq_sh, size); p.y[1] = tensor(dk, dk_st, dk_sh, size);
  hipStream_t st = (hipStream_t)stream;
  int blocks = 0;                                // no tokens: dw = 0, written by the reduction below
  if (tokens && heads + kv_heads) {
    for (int n = 0; n < 2; ++n)
      if ((normalize && !tensor_ok(p.x[n], tokens, p.heads[n], size)) || !tensor_ok(p.y[n], tokens, p.heads[n], size) || !tensor_ok(p.g[n], tokens, p.heads[n], size)) return DH_ERR_ARG;
    if (!normalize) { p.x[0] = p.g[0]; p.x[1] = p.g[1]; }
    p.part = want_w ? (float*)workspace : nullptr;
    const int rr = run(p, dtype, interleaved, normalize, true, &blocks, st);
    if (rr != DH_OK) return rr;
  }
  if (want_w) {
    hipLaunchKernelGGL(rope_dw_kernel, dim3((2 * head_dim + 7) / 8), dim3(256), 0, st, (const float*)workspace, blocks, head_dim, dq_weight, dk_weight, w_dtype);
    DH_LAUNCH_CHECK();
  }
  return DH_OK;
}
