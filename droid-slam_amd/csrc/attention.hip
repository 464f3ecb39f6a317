// Softmax attention over packed sequences of keyframe tokens, forward and backward (gfx950).
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s q_i.k_j - lse_i),  lse_i = log sum_j exp(s q_i.k_j)        over the keys j that row i sees
//   dV_j = sum_i p_ij dO_i,  dS_ij = p_ij (dO_i.v_j - delta_i),  delta_i = dO_i.o_i,  dQ_i = s sum_j dS_ij k_j,  dK_j = s sum_i dS_ij q_i
//
// Rows.  The `group` query heads that share a key head are rows of the same tile: row r = token r / group, head r % group.  Keys and
// values are then read once for the whole group, a single query of 8 heads still fills a quarter of a 32-row tile, and the gradient of a
// shared key head is summed inside one workgroup.
//
// Products.  v_mfma_f32_32x32x16 with the tile transposed: S^T = K Q^T has one row (query) per lane and 16 keys in its registers, so the
// softmax statistics are in-lane reductions plus one exchange between the wave's halves, and P^T is already the B operand of
// O^T = V^T P^T: no trip through LDS.  Register i of lane l holds key 8 (i / 4) + 4 (l / 32) + i % 4 of its 32-key block; a B operand
// wants 8 consecutive k per lane, which is met by giving A and B the same permutation of the 16 keys of a step (a sum over keys does not
// care): the transposed reads of V (ds_read_b64_tr_b16: 4 keys x 16 channels per 16 lanes) fetch keys 4 (l / 32) + {0..3, 8..11}.
//
// Memory.  64-row tiles arrive by LDS-DMA (buffer_load_dwordx4 ... lds) in two buffers, the next tile under the current one's products;
// rows behind the end and channels behind head_dim are out of the buffer's range and arrive as zeros.  The 16-byte chunks of a row are
// stored at chunk ^ swz(row): sixteen consecutive rows at one chunk (the K operand) and four consecutive rows at four (half a wave's transposed
// read) fall on different banks.
//
// Precision.  Products of 16-bit operands accumulate in 32 bits; scores, statistics, p, dP, delta and all accumulators are 32-bit.
// p and dS are rounded (to nearest) to the inputs' type as operands of the second product: their relative error is the same half step
// that the rounding of the result has, and averages over the keys; gradients are some 1.45 times as far from 64 bits as 32-bit sums rounded once
// would be (results 1.0 to 1.1 times).  delta is a difference of large sums where the keys agree: it is formed
// from o and what its rounding left behind (o_low; one more write and read of o's size), else dQ is off by 1.3 times as much.
#include "common.h"
#include <algorithm>
#include <limits.h>
#include <math.h>
#include <string.h>
#include <type_traits>

namespace {
using namespace dh;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;

struct F16 {
  using V8 = f16x8;
  // p ~ 1 / (keys) and dS are lifted by 2^4 before they are rounded: 1 / 262144 is still a normal number.  A dS has no bound: see Fit.
  static constexpr int LIFT = 4;
  // forward: p is 2^TOP where the running maximum was set, 2^(TOP + 8) at most before it is set again (2^15 fits).  Weights down to 2^-21 of the largest
  // keep fp16's precision, those below 2^-32 count as zero; with TOP = 0 that was 2^-14 and 2^-25, and a tail of thousands of them was lost together
  static constexpr float TOP = 7.f;
  static constexpr unsigned ONE = 0x3c00, INF = 0x7c00;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned pack(float x, float y) {
    f32x2 v; v.x = x; v.y = y;
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
  }
  static __device__ __forceinline__ float lo(unsigned u) { return (float)__builtin_bit_cast(f16x2, u).x; }
  static __device__ __forceinline__ float hi(unsigned u) { return (float)__builtin_bit_cast(f16x2, u).y; }
};
struct BF16 {
  using V8 = bf16x8;
  static constexpr int LIFT = 0;                 // bf16 has the exponent range of fp32
  static constexpr float TOP = 0.f;
  static constexpr unsigned ONE = 0x3f80, INF = 0x7f80;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned pack(float x, float y) {
    f32x2 v; v.x = x; v.y = y;
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
  }
  static __device__ __forceinline__ float lo(unsigned u) { return __uint_as_float(u << 16); }
  static __device__ __forceinline__ float hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
};

constexpr int BN = 64;                           // rows of an LDS tile
constexpr unsigned OUT_OF_RANGE = 0x80000000u;   // byte offset behind every buffer: such lanes of an LDS-DMA write zeros
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float M_FLOOR = -3e38f;                // start of the running maximum: finite, so that a row without keys makes no inf - inf

struct Item { int q_start, q_len, k_start, k_len, first, begin, end, slot; };   // the plan's record, see dh_attn_plan

struct View { const char* p; long st, sh; };     // base, bytes between tokens, bytes between heads

struct Params {
  View q, k, v, o, g;                            // o: the forward's output; g: its gradient
  View dq, dk, dv;
  char* low;                                     // [q_rows, heads, dim] what the rounding of o left behind, or nothing
  float* lse;                                    // [q_rows, heads]
  float* delta;                                  // backward, three of [q_rows, heads]: -delta, and what p is made from: exponent m, factor w
  long row_values;                               // (rows of the plan) * heads: from one of them to the next
  float* part;                                   // split rows: [slot, kv_heads, rows, DP] and behind them [slot, kv_heads, rows, 2]
  const Item* items;
  long n_slots;
  int blocks, clear_q, clear_k;                  // workgroups of work items; from there on: rows [clear_q, q_rows) / [clear_k, k_rows) are cleared
  int kv_heads, group, heads, dim, block, q_rows, k_rows;
  int plan_q_rows, plan_k_rows;                  // the rows that the plan's sequences have: what the workspaces are laid out for
  float c;                                       // scale * log2(e)
  float scale;
};

template <int DP> struct Geo {
  static constexpr int ROWB = DP * 2, CH = DP / 8, TILEB = BN * ROWB;
  static __device__ __forceinline__ int swz(int r) {
    const int low = (r >> 3) & 1;
    if constexpr (DP == 128) return ((r & 3) << 2) | (((r >> 2) & 1) << 1) | low;
    else if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | low;
    else return (((r >> 2) & 1) << 1) | low;
  }
};

__device__ __forceinline__ long uniform(long x) {
  return (long)(((unsigned long)(unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned long)x >> 32)) << 32) |
                (unsigned)__builtin_amdgcn_readfirstlane((int)x));
}

// the buffer of `bytes` bytes from `p` on (raw); both uniform
__device__ __forceinline__ i32x4 buffer_at(const char* p, unsigned bytes) {
  const unsigned long a = (unsigned long)p;
  i32x4 s;
  s.x = __builtin_amdgcn_readfirstlane((int)a);
  s.y = __builtin_amdgcn_readfirstlane((int)(a >> 32) & 0xffff);
  s.z = __builtin_amdgcn_readfirstlane((int)bytes);
  s.w = 0x00027000;
  return s;
}

// lane l copies 16 bytes at buffer + voff (per lane) to LDS address lds + 16 l; zeros where voff is out of range.  m0 is not kept: the compiler
// has no use for it in these kernels (build.py looks at the generated code), and saving it costs two more instructions a chunk.
__device__ __forceinline__ void dma16(i32x4 buffer, unsigned voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(voff), "s"(buffer), "s"(lds) : "memory");
}
// keeps a branch a branch: without it the selects of masked tiles are executed (and waited for) in every tile
#define RARE_BRANCH() asm volatile("")
// all but the last `LEFT` DMA instructions of this wave have arrived
template <int LEFT, bool BARRIER> __device__ __forceinline__ void dma_wait() {
  if constexpr (BARRIER) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
  else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
}
#define DMA_WAIT_BARRIER() asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory")

// One tensor's tiles of ROWS rows through LDS-DMA by NW waves.  Tile row x is token x / group (from the tile's first token on) and head
// x % group.  Rows that do not exist are behind the buffer's end (BY_END: keys, one row a token, rows at least as far apart as they are long:
// the host sees to it), or get an offset that is (heads may be further apart than tokens).
template <int DP, int NW, int ROWS, bool BY_END> struct TileLoader {
  using G = Geo<DP>;
  static constexpr int PER = (ROWS * G::CH + NW * 64 - 1) / (NW * 64);       // 16-byte chunks a thread
  static constexpr int STEP = NW * 64 / G::CH;                               // rows between two of them
  unsigned voff[PER];
  __device__ __forceinline__ void init(const View& t, int dim, int group, int rows) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int lin = i * NW * 64 + threadIdx.x, r = lin / G::CH, c = (lin % G::CH) ^ G::swz(r), tok = r / group;
      voff[i] = r < rows && c * 8 < dim ? (unsigned)(tok * t.st + (r - tok * group) * t.sh + c * 16) : OUT_OF_RANGE;
    }
  }
  // `rows`: tile rows that exist (BY_END: `stride` bytes apart and `size` bytes long)
  __device__ __forceinline__ void issue(const char* tile, int rows, unsigned stride, unsigned size, unsigned lds) const {
    const i32x4 buffer = buffer_at(tile, !BY_END ? 0x7fffffffu : rows > 0 ? (unsigned)(min(rows, ROWS) - 1) * stride + size : 0u);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = threadIdx.x / G::CH;
    if (NW * 64 > ROWS * G::CH && wave * 64 >= ROWS * G::CH) return;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      dma16(buffer, BY_END || r + i * STEP < rows ? voff[i] : OUT_OF_RANGE, lds + (i * NW + wave) * 1024);
  }
};

// operand rows 32 b .. 32 b + 31 of a tile, channels 16 s + 8 (l / 32) ..: A or B operand of a product over the channels
template <int DP> __device__ __forceinline__ u32x4 frag(const lds_char* tile, int b, int s, int lane) {
  using G = Geo<DP>;
  const int r = lane & 31;
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(tile + (b * 32 + r) * G::ROWB + (((2 * s + (lane >> 5)) ^ G::swz(r)) << 4));
}
// transposed operand: channel 32 mb + l % 32, tile rows 32 b + 16 ks + 4 (l / 32) + {0..3, 8..11}
template <int DP> __device__ __forceinline__ u32x4 frag_t(const lds_char* tile, int b, int ks, int mb, int lane) {
  using G = Geo<DP>;
  const int x = lane & 15, g = (lane >> 4) & 1, half = lane >> 5;
  u32x2 part[2];
#pragma unroll
  for (int jj = 0; jj < 2; ++jj) {
    const int r = 8 * jj + 4 * half + (x >> 2);                              // (+ 32 b + 16 ks: no bit that swz looks at)
    const int c = (2 * (2 * mb + g) + ((x & 3) >> 1)) ^ G::swz(r);
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    part[jj] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_i16x4*)(tile + (b * 32 + ks * 16 + r) * G::ROWB + c * 16 + (x & 1) * 8)));
  }
  u32x4 v; v.x = part[0].x; v.y = part[0].y; v.z = part[1].x; v.w = part[1].y;
  return v;
}

__device__ __forceinline__ float other_half(float v) {                       // the value of lane l ^ 32
  auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? x[0] : x[1]);
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// token i of a sequence sees its first keys_seen keys: all, or up to the end of the block of `block` keys that the token stands in, the last
// token standing at the last key
__host__ __device__ __forceinline__ int keys_seen(int i, int q_len, int k_len, int block) {
  if (block == 0) return k_len;
  const int at = i + (k_len - q_len);                                        // lengths and block are at most 2^30
  if (at < 0) return 0;
  const unsigned e = ((unsigned)at / (unsigned)block + 1) * (unsigned)block;
  return e < (unsigned)k_len ? (int)e : k_len;
}

// what a row's sum is multiplied by: 1 / l, and zero where nothing is seen.  Where something is, l = 0 says that every score is -inf (a maximum's own p
// is one): there is no softmax of that
__device__ __forceinline__ float row_factor(float l, int seen) { return seen <= 0 ? 0.f : l == 0.f ? NAN : 1.f / l; }

__device__ __forceinline__ bool item_ok(const Item& it, const Params& p) {   // (holds for every item of a plan with the info it came with)
  return it.q_start >= 0 && it.q_len >= 0 && it.k_start >= 0 && it.k_len >= 0 && it.first >= 0 && it.begin >= 0 &&
         (long)it.q_start + it.q_len <= p.plan_q_rows && (long)it.k_start + it.k_len <= p.plan_k_rows;
}

// acc += v^T p over 16 keys of which a row sees those below `lim` (lane's keys: from `key` on 4, and 4 more from key + 8 on).  p is 0 where a
// key is not seen, and here that also holds for a v that is not finite: such v are left out of the product and added to the rows that see them.
template <typename T> __device__ __forceinline__ void add_seen(f32x16& acc, u32x4 v, u32x4 p, int key, int lim) {
  u32x4 kind[3], seen;                           // 1 where v is +inf, -inf, NaN
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int at = key + 2 * (j & 1) + 8 * (j >> 1);
    seen[j] = (at < lim ? T::ONE : 0u) | (at + 1 < lim ? T::ONE << 16 : 0u);
    const unsigned x[2] = {v[j] & 0xffffu, v[j] >> 16};
    unsigned keep = 0u, k0 = 0u, k1 = 0u, k2 = 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned size = x[h] & 0x7fffu, one = T::ONE << (16 * h);
      keep |= (size < T::INF ? x[h] : 0u) << (16 * h);
      k0 |= x[h] == T::INF ? one : 0u;
      k1 |= x[h] == (T::INF | 0x8000u) ? one : 0u;
      k2 |= size > T::INF ? one : 0u;
    }
    v[j] = keep; kind[0][j] = k0; kind[1][j] = k1; kind[2][j] = k2;
  }
  acc = T::mfma(v, p, acc);
#pragma unroll
  for (int n = 0; n < 3; ++n) {
    f32x16 c;
#pragma unroll
    for (int i = 0; i < 16; ++i) c[i] = 0.f;
    c = T::mfma(kind[n], seen, c);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c[i] > 0.f) acc[i] += n == 0 ? INFINITY : n == 1 ? -INFINITY : NAN;
  }
}

// workgroups behind the work items: rows [from, to) of a dense or strided result become zero
template <int THREADS> __device__ __forceinline__ void clear_rows(const View& t, int from, int to, int heads, int dim, int part, int parts) {
  const long n = (long)(to - from) * heads * (dim / 8);
  for (long i = (long)part * THREADS + threadIdx.x; i < n; i += (long)parts * THREADS) {
    const long c = i % (dim / 8), r = i / (dim / 8);
    *reinterpret_cast<u32x4*>(const_cast<char*>(t.p) + (from + r / heads) * t.st + r % heads * t.sh + c * 16) = u32x4{0u, 0u, 0u, 0u};
  }
}
constexpr int CLEAR_BYTES = 1 << 15;             // a workgroup's share

// ------------------------------------------------------------------------------------------------------------- forward
// One workgroup: NW x 32 rows (NW * 32 / group tokens) of one key head over the keys [begin, end) of its sequence.  Running maximum and sum
// per row; the accumulator is only rescaled when a maximum grew by more than 2^8 (p <= 2^(TOP + 8) until then: exact in 32 bits, and a 16-bit p
// keeps its relative precision, in fp16 down to 2^-21 of the largest).  slot >= 0: the row range is split over the keys, unnormalised sums go to the workspace for attn_join.
// Bound by the matrix cores at the power limit (128 channels: 1.04 .. 1.11 PFLOP/s by card on 19200 tokens, the library's large product 1.25), by the vector
// units at 64 channels (0.72 on packed clips, whose longest walks of 69 tiles also outlast a mean of 27: see dh_attn_plan).
// How the keys come in: 64 keys a tile, one tile ahead; a lone wave (few rows, bound by memory: 82 us for 32 queries over 358 MB of keys, 4.4 TB/s)
// takes 32 and keeps two tiles on their way in 48 KB, three waves a CU (90 us; with the same plan, two or four stages and as many waves as fit: 99, 95).
template <int NW> struct Walk { static constexpr int BLOCKS = NW == 1 ? 1 : 2, STAGES = NW == 1 ? 3 : 2; };

template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 1 ? 1 : DP == 128 ? 2 : 3) void attn_fwd_kernel(const Params p) {
  using G = Geo<DP>;
  constexpr int KB = Walk<NW>::BLOCKS, TK = KB * 32, ST = Walk<NW>::STAGES, TB = TK * G::ROWB;
  __shared__ __attribute__((aligned(1024))) char smem[ST * 2 * TB];          // [stage][K, V]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x >= p.blocks) {
    const int part = blockIdx.x - p.blocks, parts = gridDim.x - p.blocks;
    clear_rows<NW * 64>(p.o, p.clear_q, p.q_rows, p.heads, p.dim, part, parts);
    for (long i = (long)p.clear_q * p.heads + part * NW * 64 + threadIdx.x; i < (long)p.q_rows * p.heads; i += parts * NW * 64) p.lse[i] = -INFINITY;
    return;
  }
  const Item it = p.items[blockIdx.x / p.kv_heads];
  const int hk = blockIdx.x % p.kv_heads;
  if (!item_ok(it, p) || it.first >= it.q_len || it.slot >= p.n_slots) return;
  const int row = wave * 32 + (lane & 31), tpt = NW * 32 / p.group;          // tokens a tile
  const int tok = it.first + row / p.group, head = hk * p.group + row % p.group;
  const bool valid = row < tpt * p.group && tok < it.q_len;
  const int key_end = min(it.end, it.k_len);
  const int lim = valid ? min(keys_seen(tok, it.q_len, it.k_len, p.block), key_end) : key_end;
  const int wmin = wave_min(lim);

  u32x4 qf[DP / 16];
  {
    const char* qp = p.q.p + (long)(it.q_start + (valid ? tok : it.first)) * p.q.st + (long)(valid ? head : hk * p.group) * p.q.sh;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      qf[s] = d < p.dim ? *reinterpret_cast<const u32x4*>(qp + d * 2) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x16 acc[DP / 32];
  float m, l;                                                                // l: this half's keys only
  TileLoader<DP, NW, TK, true> lk, lv;
  lk.init(p.k, p.dim, 1, TK);
  lv.init(p.v, p.dim, 1, TK);
  const char* kp = p.k.p + uniform((long)(it.k_start + it.begin) * p.k.st + (long)hk * p.k.sh);
  const char* vp = p.v.p + uniform((long)(it.k_start + it.begin) * p.v.st + (long)hk * p.v.sh);
  lds_char* const lds = (lds_char*)smem;
  const unsigned lds0 = (unsigned)(unsigned long)lds;
  const int tiles = (key_end - it.begin + TK - 1) / TK;
  // the next K / V tile; behind the last one nothing is read, zeros go to a stage nobody reads
  const unsigned k_st = (unsigned)p.k.st, v_st = (unsigned)p.v.st;
  const char *k_next, *v_next;
  int k_left, v_left, k_to, v_to;
  auto issue_k = [&]() {
    lk.issue(k_next, k_left, k_st, p.dim * 2, lds0 + k_to);
    k_next += (long)TK * k_st;
    k_left -= TK;
    k_to = k_to == (ST - 1) * 2 * TB ? 0 : k_to + 2 * TB;
  };
  auto issue_v = [&]() {
    lv.issue(v_next, v_left, v_st, p.dim * 2, lds0 + TB + v_to);
    v_next += (long)TK * v_st;
    v_left -= TK;
    v_to = v_to == (ST - 1) * 2 * TB ? 0 : v_to + 2 * TB;
  };
  const auto k_tile = [&](int t) { return lds + t % ST * 2 * TB; };
  const auto v_tile = [&](int t) { return lds + t % ST * 2 * TB + TB; };

  // the scores of 32 keys: block b of a K tile
  auto scores = [&](const lds_char* kt, int b) {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = T::mfma(frag<DP>(kt, b, ks, lane), qf[ks], s);
    return s;
  };
  // hides what a row does not see and keeps p at or below 2^(TOP + 8), looking at the exponent that p gets (at scores of 10^8 the maximum's own
  // rounding is +- 8: the new one is formed in one step).  Each half of the wave looks at its own keys of a row; only where one of
  // them found a maximum that is too large the halves agree on a new one.
  auto settle = [&](f32x16& s, int n0) {
    if (n0 + 32 > wmin) {
      RARE_BRANCH();
      const int end = lim - n0 - 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + (i & 3) >= end) s[i] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    if (__any(fmaf(mx, p.c, -m) > T::TOP + 8.f)) {
      RARE_BRANCH();
      mx = fmaxf(mx, other_half(mx));
      const float mn = fmaf(mx, p.c, -m) > T::TOP + 8.f ? fmaf(mx, p.c, -T::TOP) : m, a = exp2_fast(m - mn);         // (a row's bits do not depend on its neighbours)
      m = mn;
      l *= a;
#pragma unroll
      for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[mb][i] *= a;
    }
  };
  auto soften = [&](f32x16& s, u32x4 (&pf)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = exp2_fast(fmaf(s[i], p.c, -m));
      l += s[i];
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int j = 0; j < 4; ++j) pf[ks][j] = T::pack(s[8 * ks + 2 * j], s[8 * ks + 2 * j + 1]);
  };
  auto walk = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
    m = M_FLOOR;
    l = 0.f;
    k_next = kp; v_next = vp;
    k_left = v_left = key_end - it.begin;
    k_to = v_to = 0;
#pragma unroll
    for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mb][i] = 0.f;
    auto add = [&](const lds_char* vt, int b, u32x4 (&pf)[2], int n0) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int mb = 0; mb < DP / 32; ++mb) {
          const u32x4 vf = frag_t<DP>(vt, b, ks, mb, lane);
          if (CAREFUL && n0 + 32 > wmin) add_seen<T>(acc[mb], vf, pf[ks], n0 + ks * 16 + 4 * (lane >> 5), lim);
          else acc[mb] = T::mfma(vf, pf[ks], acc[mb]);
        }
    };
    u32x4 pf[2];
    if constexpr (NW == 1) {
      for (int t = 0; t < ST - 1; ++t) { issue_k(); issue_v(); }
      for (int t = 0; t < tiles; ++t) {
        dma_wait<(ST - 2) * 2 * TileLoader<DP, NW, TK, true>::PER, false>();       // (the stages behind tile t may still be on their way)
        issue_k();
        issue_v();
        const int n0 = it.begin + t * TK;
        f32x16 s = scores(k_tile(t), 0);
        settle(s, n0);
        soften(s, pf);
        add(v_tile(t), 0, pf, n0);
      }
    } else if (tiles > 0) {
      // The next block's scores are formed (matrix cores) while the exponentials of this one are (vector units); so K runs ahead of V by a
      // tile, and one barrier a tile serves both: before it K t and V t - 1 were read for the last time, behind it K t + 1 and V t are there.
      issue_k();
      dma_wait<0, true>();
      issue_v();
      issue_k();
      f32x16 s = scores(k_tile(0), 0);
      for (int t = 0; t < tiles; ++t) {
        const int n0 = it.begin + t * TK;
        settle(s, n0);
        f32x16 s1 = scores(k_tile(t), 1);
        soften(s, pf);
        dma_wait<0, true>();
        issue_v();
        issue_k();
        add(v_tile(t), 0, pf, n0);
        settle(s1, n0 + 32);
        s = scores(k_tile(t + 1), 0);                                        // (behind the last tile: zeros, not used)
        soften(s1, pf);
        add(v_tile(t), 1, pf, n0 + 32);
      }
    }
    dma_wait<0, (NW > 1)>();                                                 // (nothing may arrive later)
  };
  walk(std::false_type());
  // A value that is not finite makes 0 * v of the rows that do not see it NaN.  Only then the workgroup walks a second time.
  bool odd = false;
#pragma unroll
  for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
    for (int i = 0; i < 16; ++i) odd |= acc[mb][i] != acc[mb][i];
  odd = __any(odd && valid);
  if (NW > 1) {
    int* flag = reinterpret_cast<int*>(smem);
    __syncthreads();
    if (lane == 0) flag[wave] = odd;
    __syncthreads();
    odd = false;
#pragma unroll
    for (int i = 0; i < NW; ++i) odd |= flag[i] != 0;
    __syncthreads();
  }
  if (odd) walk(std::true_type());
  l += other_half(l);
  if (it.slot >= 0) {
    const long at = (((long)it.slot * p.kv_heads + hk) * (NW * 32) + row);
    float* po = p.part + at * DP;
#pragma unroll
    for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        f32x4 v; v.x = acc[mb][4 * i4]; v.y = acc[mb][4 * i4 + 1]; v.z = acc[mb][4 * i4 + 2]; v.w = acc[mb][4 * i4 + 3];
        *reinterpret_cast<f32x4*>(po + mb * 32 + 8 * i4 + 4 * (lane >> 5)) = v;
      }
    if (lane < 32) {
      float* pm = p.part + p.n_slots * p.kv_heads * (NW * 32) * DP + at * 2;
      pm[0] = m;
      pm[1] = l;
    }
    return;
  }
  if (!valid) return;
  const float inv = row_factor(l, lim);
  char* op = const_cast<char*>(p.o.p) + (long)(it.q_start + tok) * p.o.st + (long)head * p.o.sh;
  char* lp = p.low + ((long)(it.q_start + tok) * p.heads + head) * p.dim * 2;
#pragma unroll
  for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int d = mb * 32 + 8 * i4 + 4 * (lane >> 5);
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = acc[mb][4 * i4 + j] * inv;
      const u32x2 v = {T::pack(x[0], x[1]), T::pack(x[2], x[3])};
      if (d >= p.dim) continue;
      *reinterpret_cast<u32x2*>(op + d * 2) = v;
      if (p.low) *reinterpret_cast<u32x2*>(lp + d * 2) = u32x2{T::pack(x[0] - T::lo(v.x), x[1] - T::hi(v.x)), T::pack(x[2] - T::lo(v.y), x[3] - T::hi(v.y))};
    }
  if (lane < 32) p.lse[(long)(it.q_start + tok) * p.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// joins the parts of split rows: items {q_start, q_len, -, -, first, first slot, slots, -}; one 32-lane half of a wave per row
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(const Params p, int rows) {
  const Item it = p.items[blockIdx.y / p.kv_heads];
  const int hk = blockIdx.y % p.kv_heads;
  const int row = blockIdx.x * 8 + threadIdx.x / 32, x = threadIdx.x & 31;
  const int tok = it.first + row / p.group, head = hk * p.group + row % p.group;
  if (row >= rows / p.group * p.group || tok >= it.q_len || !item_ok(it, p) || (long)it.begin + it.end > p.n_slots) return;   // (whole halves of waves)
  // lane x holds the statistics of part x (x + 32, ...); all loads of a loop are independent of each other
  const float* pm = p.part + p.n_slots * p.kv_heads * rows * DP;
  const auto at = [&](int i) { return ((long)(it.begin + i) * p.kv_heads + hk) * rows + row; };
  float m = M_FLOOR, l = 0.f, acc[DP / 32];
  for (int i = x; i < it.end; i += 32) m = fmaxf(m, pm[at(i) * 2]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
#pragma unroll
  for (int k = 0; k < DP / 32; ++k) acc[k] = 0.f;
  for (int i0 = 0; i0 < it.end; i0 += 32) {
    const int n = min(32, it.end - i0);
    const float w = x < n ? exp2f(pm[at(i0 + x) * 2] - m) : 0.f;
    if (x < n) l += w * pm[at(i0 + x) * 2 + 1];
    for (int j0 = 0; j0 < n; j0 += 8) {
      float v[8][DP / 32];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int k = 0; k < DP / 32; ++k) v[j][k] = p.part[at(i0 + min(j0 + j, n - 1)) * DP + k * 32 + x];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = __shfl(w, (threadIdx.x & 32) + j0 + j, 64);          // (0 from n on)
        if (j0 + j < n) {
#pragma unroll
          for (int k = 0; k < DP / 32; ++k) acc[k] += a * v[j][k];
        }
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
  const float inv = row_factor(l, keys_seen(tok, it.q_len, it.k_len, p.block));
  unsigned short* op = reinterpret_cast<unsigned short*>(const_cast<char*>(p.o.p) + (long)(it.q_start + tok) * p.o.st + (long)head * p.o.sh);
#pragma unroll
  for (int k = 0; k < DP / 32; ++k)
    if (k * 32 + x < p.dim) {
      const unsigned u = T::pack(acc[k] * inv, 0.f);
      op[k * 32 + x] = (unsigned short)u;
      if (p.low) reinterpret_cast<unsigned short*>(p.low)[((long)(it.q_start + tok) * p.heads + head) * p.dim + k * 32 + x] = (unsigned short)T::pack(acc[k] * inv - T::lo(u), 0.f);
    }
  if (x == 0) p.lse[(long)(it.q_start + tok) * p.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// ------------------------------------------------------------------------------------------------------------ backward
// fp16 holds numbers up to 65504 where dS may be any size, however small the gradients that it sums to (a loss scale makes such dO).  So the
// columns of dS^T that a lane's sum is made of (a row's for dQ, a key's for dK) get a power of two of their own when one of them passes 2^15: it is
// taken out of the sum again at the end.  Until then there is only the largest |dS| to look at (some 10 instructions to 16 scores; training clips, fp16: 169 -> 175 us).
template <typename T, int N> struct Fit {
  float factor = 1.f, most = 32768.f;
  // before s is packed; both halves of the wave hold parts of the same column
  __device__ __forceinline__ void operator()(f32x16& s, f32x16 (&acc)[N]) {
    if constexpr (T::LIFT != 0) {
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(s[i]));
      if (__any(mx > most)) {
        RARE_BRANCH();
        mx = fmaxf(mx, other_half(mx));
        // the largest becomes 2^13 .. 2^14: two more doublings fit before the sums are scaled again
        const float to = mx * factor > 32768.f ? ldexpf(1.f, 14 - __builtin_amdgcn_frexp_expf(mx)) : factor, a = to / factor;
        factor = to;
        most = to < 1.f ? -1.f : 32768.f;                                    // from now on every s is scaled
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] *= to;
#pragma unroll
        for (int mb = 0; mb < N; ++mb)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[mb][i] *= a;
      }
    }
  }
};

// dQ: the forward's walk over the keys with dO next to Q.  S^T and dP^T = V dO^T give dS^T in the layout of a B operand; the K tile is
// read a second time transposed for dQ^T = K^T dS^T.  Split as the forward is; 1.13 .. 1.18 PFLOP/s (by card) on a training window of 14400 tokens
// (128 channels).
// p.  lse has 32 bits: at scores of 10^6 its last bit is 4 % of p, at 10^8 a factor of 250.  So it only says where p is about 1: the walk forms
// p' = exp2(s c - m), m from lse, and the sum l' of the p' it formed; dQ is divided by l', and attn_dkv_kernel takes p = p' w, w = 1 / l', from the
// same m and the same bits of s.  m is lowered by what lse can be off (its three roundings and two constants: 4.5 2^-24 of itself), so that l' is 1 at
// least: at scores of 10^8 it may reach 2^80, which only fp16 minds (Fit).  The sum costs what the products save that start at -delta instead of 0.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, DP == 128 ? 2 : 3) void attn_dq_kernel(const Params p) {
  using G = Geo<DP>;
  __shared__ __attribute__((aligned(1024))) char smem[4 * G::TILEB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x >= p.blocks) {
    clear_rows<NW * 64>(p.dq, p.clear_q, p.q_rows, p.heads, p.dim, blockIdx.x - p.blocks, gridDim.x - p.blocks);
    return;
  }
  const Item it = p.items[blockIdx.x / p.kv_heads];
  const int hk = blockIdx.x % p.kv_heads;
  if (!item_ok(it, p) || it.first >= it.q_len || it.slot >= p.n_slots) return;
  const int row = wave * 32 + (lane & 31), tpt = NW * 32 / p.group;
  const int tok = it.first + row / p.group, head = hk * p.group + row % p.group;
  const bool valid = row < tpt * p.group && tok < it.q_len;
  const int key_end = min(it.end, it.k_len);
  const int lim = valid ? min(keys_seen(tok, it.q_len, it.k_len, p.block), key_end) : key_end;
  const int wmin = wave_min(lim), wmax = wave_max(valid ? lim : 0);

  u32x4 qf[DP / 16], gf[DP / 16];
  const long t_ = it.q_start + (valid ? tok : it.first), h_ = valid ? head : hk * p.group;
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * (lane >> 5);
    const bool in = d < p.dim;
    qf[s] = in ? *reinterpret_cast<const u32x4*>(p.q.p + t_ * p.q.st + h_ * p.q.sh + d * 2) : u32x4{0u, 0u, 0u, 0u};
    gf[s] = in ? *reinterpret_cast<const u32x4*>(p.g.p + t_ * p.g.st + h_ * p.g.sh + d * 2) : u32x4{0u, 0u, 0u, 0u};
    const u32x4 of = in ? *reinterpret_cast<const u32x4*>(p.o.p + t_ * p.o.st + h_ * p.o.sh + d * 2) : u32x4{0u, 0u, 0u, 0u};
    const u32x4 rf = in && p.low ? *reinterpret_cast<const u32x4*>(p.low + ((t_ * p.heads + h_) * p.dim + d) * 2) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 4; ++j) delta += T::lo(gf[s][j]) * (T::lo(of[j]) + T::lo(rf[j])) + T::hi(gf[s][j]) * (T::hi(of[j]) + T::hi(rf[j]));
  }
  delta += other_half(delta);
  const float lse2 = p.lse[t_ * p.heads + h_] * LOG2E;
  const float m = lse2 == -INFINITY ? 0.f : lse2 - fabsf(lse2) * 0x1.2p-22f - T::LIFT;                 // (finite where nothing is seen)
  if (valid && lane < 32 && it.begin == 0) {                                 // (the first of a split walk)
    p.delta[t_ * p.heads + h_] = -delta;
    p.delta[t_ * p.heads + h_ + p.row_values] = m;
  }
  float l = 0.f;                                                             // this half's keys only

  f32x16 acc[DP / 32];
#pragma unroll
  for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[mb][i] = 0.f;
  Fit<T, DP / 32> fit;
  TileLoader<DP, NW, BN, true> lk, lv;
  lk.init(p.k, p.dim, 1, BN);
  lv.init(p.v, p.dim, 1, BN);
  const char* kp = p.k.p + uniform((long)(it.k_start + it.begin) * p.k.st + (long)hk * p.k.sh);
  const char* vp = p.v.p + uniform((long)(it.k_start + it.begin) * p.v.st + (long)hk * p.v.sh);
  lds_char* const lds = (lds_char*)smem;
  const unsigned lds0 = (unsigned)(unsigned long)lds;
  const int tiles = (key_end - it.begin + BN - 1) / BN;
  int left = key_end - it.begin;
  const unsigned k_st = (unsigned)p.k.st, v_st = (unsigned)p.v.st;
  auto issue = [&](int t) {                                                  // in order
    const unsigned to = lds0 + (t & 1) * 2 * G::TILEB;
    lk.issue(kp, left, k_st, p.dim * 2, to);
    lv.issue(vp, left, v_st, p.dim * 2, to + G::TILEB);
    kp += (long)BN * k_st;
    vp += (long)BN * v_st;
    left -= BN;
  };
  if (tiles > 0) issue(0);
  for (int t = 0; t < tiles; ++t) {
    DMA_WAIT_BARRIER();
    if (t + 1 < tiles) issue(t + 1);
    const int n0 = it.begin + t * BN;
    if (n0 >= wmax) continue;
    const lds_char* kt = lds + (t & 1) * 2 * G::TILEB;
    const lds_char* vt = kt + G::TILEB;
    const bool masked = n0 + BN > wmin;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = -delta; }
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        s = T::mfma(frag<DP>(kt, b, ks, lane), qf[ks], s);
        dp = T::mfma(frag<DP>(vt, b, ks, lane), gf[ks], dp);
      }
      if (masked) {
        RARE_BRANCH();
        const int end = lim - n0 - 4 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (b * 32 + 8 * (i / 4) + (i & 3) >= end) { s[i] = -INFINITY; dp[i] = 0.f; }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = exp2_fast(fmaf(s[i], p.c, -m));
        l += s[i];
        s[i] *= dp[i];
      }
      fit(s, acc);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x4 df;
#pragma unroll
        for (int j = 0; j < 4; ++j) df[j] = T::pack(s[8 * ks + 2 * j], s[8 * ks + 2 * j + 1]);
#pragma unroll
        for (int mb = 0; mb < DP / 32; ++mb) acc[mb] = T::mfma(frag_t<DP>(kt, b, ks, mb, lane), df, acc[mb]);
      }
    }
  }
  l += other_half(l);
  if (it.slot >= 0) {
    const long at = ((long)it.slot * p.kv_heads + hk) * (NW * 32) + row;
    float* out = p.part + at * DP;
    const float f = 1.f / fit.factor;
    if (lane < 32) p.part[p.n_slots * p.kv_heads * (NW * 32) * DP + at] = l;
#pragma unroll
    for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4)
        *reinterpret_cast<f32x4*>(out + mb * 32 + 8 * i4 + 4 * (lane >> 5)) = f32x4{acc[mb][4 * i4] * f, acc[mb][4 * i4 + 1] * f, acc[mb][4 * i4 + 2] * f, acc[mb][4 * i4 + 3] * f};
    return;
  }
  if (!valid) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f, f = p.scale * inv / fit.factor;
  if (lane < 32) p.delta[t_ * p.heads + h_ + 2 * p.row_values] = inv * (1 << T::LIFT);
  char* op = const_cast<char*>(p.dq.p) + t_ * p.dq.st + h_ * p.dq.sh;
#pragma unroll
  for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int d = mb * 32 + 8 * i4 + 4 * (lane >> 5);
      u32x2 v;
      v.x = T::pack(acc[mb][4 * i4] * f, acc[mb][4 * i4 + 1] * f);
      v.y = T::pack(acc[mb][4 * i4 + 2] * f, acc[mb][4 * i4 + 3] * f);
      if (d < p.dim) *reinterpret_cast<u32x2*>(op + d * 2) = v;
    }
}

// adds the parts of split rows: items {q_start, q_len, -, -, first, first slot, slots, -}; a thread adds 4 channels of one row
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dq_join_kernel(const Params p) {
  const Item it = p.items[blockIdx.y / p.kv_heads];
  const int hk = blockIdx.y % p.kv_heads;
  const int at = blockIdx.x * 256 + threadIdx.x, row = at / (DP / 4), d = at % (DP / 4) * 4;
  const int tok = it.first + row / p.group, head = hk * p.group + row % p.group;
  if (row >= 128 / p.group * p.group || tok >= it.q_len || d >= p.dim || !item_ok(it, p) || (long)it.begin + it.end > p.n_slots) return;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int i = 0; i < it.end; ++i) {
    const long slot = ((long)(it.begin + i) * p.kv_heads + hk) * 128 + row;
    sum += *reinterpret_cast<const f32x4*>(p.part + slot * DP + d);
    l += p.part[p.n_slots * p.kv_heads * 128 * DP + slot];
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f, f = p.scale * inv;
  if (d == 0) p.delta[(long)(it.q_start + tok) * p.heads + head + 2 * p.row_values] = inv * (1 << T::LIFT);
  *reinterpret_cast<u32x2*>(const_cast<char*>(p.dq.p) + (long)(it.q_start + tok) * p.dq.st + (long)head * p.dq.sh + d * 2) =
      u32x2{T::pack(sum.x * f, sum.y * f), T::pack(sum.z * f, sum.w * f)};
}

// dK, dV: one workgroup holds 64 keys of one key head (128 where head_dim > 64), 32 a wave, and walks over the rows (tokens x group) that see
// them, 64 rows a tile, 32 a wave: 4 (8) waves, the two halves of the rows meet at the end.
// S = Q K^T and dP = dO V^T have one key per lane, so P and dS are B operands of dV^T = dO^T P and dK^T = Q^T dS.
// What bounds it is the wait for LDS operands, which a wave can only read ahead into registers it has: at 128 channels the two accumulators are
// 128 of 256.  With K and V in registers the kernel spilled (training window of 12 x 1200 tokens: 6.0 ms), with V in LDS it had no room to
// read ahead (2.1 ms), with both in LDS, a tile serving 8 waves, it takes 1.87 ms.  64 keys a wave (half the LDS reads, one wave a SIMD) spilled.
// slot >= 0: the walk over the rows is split, 32-bit sums go to the workspace for attn_dkv_join.
template <int DP> struct Dkv {
  static constexpr bool WIDE = DP == 128;                                    // K in LDS as well
  static constexpr int KW = WIDE ? 4 : 2, RW = 2;                            // waves along the keys / along the rows
  static constexpr int WAVES = KW * RW, KEYS = KW * 32, ROWS = RW * 32, TB = ROWS * Geo<DP>::ROWB;
  static constexpr int LDS = 4 * TB + (WIDE ? 2 : 1) * KEYS * Geo<DP>::ROWB + 7 * ROWS * 4;
};

template <typename T, int DP>
__global__ __launch_bounds__(Dkv<DP>::WAVES * 64, DP == 128 ? 2 : 3) void attn_dkv_kernel(const Params p) {
  using G = Geo<DP>;
  constexpr int TB = Dkv<DP>::TB, DKV_ROWS = Dkv<DP>::ROWS, DKV_KEYS = Dkv<DP>::KEYS, DKV_WAVES = Dkv<DP>::WAVES;
  constexpr bool WIDE = Dkv<DP>::WIDE;
  extern __shared__ __attribute__((aligned(1024))) char dyn[];               // [buffer][Q, dO], V (and K), [buffer][m, w, -delta], tokens of the rows
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % Dkv<DP>::KW, rw = (threadIdx.x >> 6) / Dkv<DP>::KW;       // 32 keys, 32 rows of a tile
  if (blockIdx.x >= p.blocks) {
    clear_rows<DKV_WAVES * 64>(p.dk, p.clear_k, p.k_rows, p.kv_heads, p.dim, blockIdx.x - p.blocks, gridDim.x - p.blocks);
    clear_rows<DKV_WAVES * 64>(p.dv, p.clear_k, p.k_rows, p.kv_heads, p.dim, blockIdx.x - p.blocks, gridDim.x - p.blocks);
    return;
  }
  const Item it = p.items[blockIdx.x / p.kv_heads];
  const int hk = blockIdx.x % p.kv_heads;
  if (!item_ok(it, p) || it.first >= it.k_len || it.slot >= p.n_slots) return;
  const int key = it.first + wave * 32 + (lane & 31);
  const bool valid = key < it.k_len;
  char* const vtile = dyn + 4 * TB;
  float* const stat = reinterpret_cast<float*>(vtile + (WIDE ? 2 : 1) * DKV_KEYS * G::ROWB);
  int* const row_tok = reinterpret_cast<int*>(stat + 6 * DKV_ROWS);
  lds_char* const lds = (lds_char*)dyn;
  const unsigned lds0 = (unsigned)(unsigned long)lds;
  {
    TileLoader<DP, DKV_WAVES, DKV_KEYS, true> l;
    l.init(p.v, p.dim, 1, DKV_KEYS);
    l.issue(p.v.p + uniform((long)(it.k_start + it.first) * p.v.st + (long)hk * p.v.sh), it.k_len - it.first, (unsigned)p.v.st, p.dim * 2, lds0 + 4 * TB);
    if (WIDE) {
      l.init(p.k, p.dim, 1, DKV_KEYS);
      l.issue(p.k.p + uniform((long)(it.k_start + it.first) * p.k.st + (long)hk * p.k.sh), it.k_len - it.first, (unsigned)p.k.st, p.dim * 2, lds0 + 4 * TB + DKV_KEYS * G::ROWB);
    }
  }
  u32x4 kf[DP / 16];
  {
    const char* kp = p.k.p + (long)(it.k_start + (valid ? key : it.k_len - 1)) * p.k.st + (long)hk * p.k.sh;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      kf[s] = d < p.dim ? *reinterpret_cast<const u32x4*>(kp + d * 2) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[mb][i] = dv[mb][i] = 0.f;
  Fit<T, DP / 32> fit;

  const int tpt = DKV_ROWS / p.group;                                        // tokens a tile
  TileLoader<DP, DKV_WAVES, DKV_ROWS, false> lq, lg;
  lq.init(p.q, p.dim, p.group, tpt * p.group);
  lg.init(p.g, p.dim, p.group, tpt * p.group);
  const int tok_end = min(it.end, it.q_len);
  const int tiles = (tok_end - it.begin + tpt - 1) / tpt;
  const char* qp = p.q.p + uniform((long)(it.q_start + it.begin) * p.q.st + (long)hk * p.group * p.q.sh);
  const char* gp = p.g.p + uniform((long)(it.q_start + it.begin) * p.g.st + (long)hk * p.group * p.g.sh);
  // A key is seen from token seen_from(key) on (what keys_seen says, solved for the token): per lane, and for the first and last key of
  // the wave.
  auto seen_from = [&](int k) { return p.block ? (int)((unsigned)k / (unsigned)p.block * (unsigned)p.block) - (it.k_len - it.q_len) : 0; };
  const int from = seen_from(key), wave_any = seen_from(it.first + wave * 32), wave_all = seen_from(min(it.first + wave * 32 + 32, it.k_len) - 1);
  // row statistics: DKV_ROWS threads hold a row of the next tile each
  const int mrow = threadIdx.x, mtok = mrow / p.group, mhead = hk * p.group + mrow % p.group;
  float r_m = 0.f, r_w = 0.f, r_delta = 0.f;
  if (mrow < DKV_ROWS) row_tok[mrow] = mtok;
  auto fetch = [&](int t) {
    if (mrow >= DKV_ROWS) return;
    const int tk = it.begin + t * tpt + mtok;
    const bool in = mrow < tpt * p.group && tk < tok_end;
    const long at = (long)(it.q_start + (in ? tk : it.begin)) * p.heads + (in ? mhead : hk * p.group);
    r_delta = in ? p.delta[at] : 0.f;
    r_m = in ? p.delta[at + p.row_values] : 0.f;
    r_w = in ? p.delta[at + 2 * p.row_values] : 0.f;                         // p = 0 in rows that do not exist
  };
  auto park = [&](int t) {
    if (mrow >= DKV_ROWS) return;
    float* f = stat + (t & 1) * 3 * DKV_ROWS + mrow;
    f[0] = r_m;
    f[DKV_ROWS] = r_w;
    f[2 * DKV_ROWS] = r_delta;
  };
  auto issue = [&](int t) {
    const unsigned to = lds0 + (t & 1) * 2 * TB;
    const int rows = min(tok_end - it.begin - t * tpt, tpt) * p.group;
    lq.issue(qp, rows, 0, 0, to);
    lg.issue(gp, rows, 0, 0, to + TB);
    qp += tpt * p.q.st;
    gp += tpt * p.g.st;
  };
  if (tiles > 0) {
    fetch(0);
    issue(0);
    park(0);
  }
  for (int t = 0; t < tiles; ++t) {
    DMA_WAIT_BARRIER();
    if (t + 1 < tiles) {
      fetch(t + 1);
      issue(t + 1);
    }
    const lds_char* qt = lds + (t & 1) * 2 * TB;
    const lds_char* gt = qt + TB;
    const lds_char* vt = lds + 4 * TB;
    const float* st = stat + (t & 1) * 3 * DKV_ROWS;
    const int first_tok = it.begin + t * tpt;
    if (first_tok + tpt > wave_any) {                                        // (else no row of the tile sees a key of the wave)
      f32x16 s, dp;
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4 from_delta = *reinterpret_cast<const f32x4*>(st + 2 * DKV_ROWS + rw * 32 + 8 * i4 + 4 * (lane >> 5));
#pragma unroll
        for (int j = 0; j < 4; ++j) { s[4 * i4 + j] = 0.f; dp[4 * i4 + j] = from_delta[j]; }
      }
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        if constexpr (WIDE) s = T::mfma(frag<DP>(qt, rw, ks, lane), frag<DP>(vt + DKV_KEYS * G::ROWB, wave, ks, lane), s);
        else s = T::mfma(frag<DP>(qt, rw, ks, lane), kf[ks], s);
        dp = T::mfma(frag<DP>(gt, rw, ks, lane), frag<DP>(vt, wave, ks, lane), dp);
      }
      const bool masked = first_tok < wave_all;
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int r = rw * 32 + 8 * i4 + 4 * (lane >> 5);
        const f32x4 m = *reinterpret_cast<const f32x4*>(st + r);
        const f32x4 w = *reinterpret_cast<const f32x4*>(st + DKV_ROWS + r);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * i4 + j;
          s[i] = exp2_fast(fmaf(s[i], p.c, -m[j])) * w[j];
          dp[i] *= s[i];
        }
        if (masked) {
          RARE_BRANCH();
          const i32x4 tok = *reinterpret_cast<const i32x4*>(row_tok + r);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (first_tok + tok[j] < from) s[4 * i4 + j] = dp[4 * i4 + j] = 0.f;
        }
      }
      fit(dp, dk);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x4 pf, df;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pf[j] = T::pack(s[8 * ks + 2 * j], s[8 * ks + 2 * j + 1]);
          df[j] = T::pack(dp[8 * ks + 2 * j], dp[8 * ks + 2 * j + 1]);
        }
#pragma unroll
        for (int mb = 0; mb < DP / 32; ++mb) {
          dv[mb] = T::mfma(frag_t<DP>(gt, rw, ks, mb, lane), pf, dv[mb]);
          dk[mb] = T::mfma(frag_t<DP>(qt, rw, ks, mb, lane), df, dk[mb]);
        }
      }
    }
    if (t + 1 < tiles) park(t + 1);                                          // (its buffer was last read before this iteration's barrier)
  }
  if (tiles == 0) DMA_WAIT_BARRIER();                                        // (V is still on its way)
  if constexpr (T::LIFT != 0) {
    const float a = 1.f / fit.factor;
#pragma unroll
    for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[mb][i] *= a;
  }
  {                                                                          // the two halves of the rows meet in LDS, where the tiles were
    static_assert(Dkv<DP>::RW == 2, "two waves to a key");
    float* sum = reinterpret_cast<float*>(dyn) + wave * (DP * 64) + lane;
    __syncthreads();
    if (rw) {
#pragma unroll
      for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
        for (int i = 0; i < 16; ++i) { sum[(mb * 32 + i) * 64] = dk[mb][i]; sum[(mb * 32 + 16 + i) * 64] = dv[mb][i]; }
    }
    __syncthreads();
    if (rw) return;
#pragma unroll
    for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) { dk[mb][i] += sum[(mb * 32 + i) * 64]; dv[mb][i] += sum[(mb * 32 + 16 + i) * 64]; }
  }
  const float fv = 1.f / (1 << T::LIFT), fk = p.scale * fv;
  if (it.slot >= 0) {
    float* out = p.part + ((((long)it.slot * p.kv_heads + hk) * DKV_KEYS) + wave * 32 + (lane & 31)) * 2 * DP;
#pragma unroll
    for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int d = mb * 32 + 8 * i4 + 4 * (lane >> 5);
        *reinterpret_cast<f32x4*>(out + d) = f32x4{dk[mb][4 * i4] * fk, dk[mb][4 * i4 + 1] * fk, dk[mb][4 * i4 + 2] * fk, dk[mb][4 * i4 + 3] * fk};
        *reinterpret_cast<f32x4*>(out + DP + d) = f32x4{dv[mb][4 * i4] * fv, dv[mb][4 * i4 + 1] * fv, dv[mb][4 * i4 + 2] * fv, dv[mb][4 * i4 + 3] * fv};
      }
    return;
  }
  if (!valid) return;
  char* kp = const_cast<char*>(p.dk.p) + (long)(it.k_start + key) * p.dk.st + (long)hk * p.dk.sh;
  char* vp = const_cast<char*>(p.dv.p) + (long)(it.k_start + key) * p.dv.st + (long)hk * p.dv.sh;
#pragma unroll
  for (int mb = 0; mb < DP / 32; ++mb)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int d = mb * 32 + 8 * i4 + 4 * (lane >> 5);
      if (d >= p.dim) continue;
      *reinterpret_cast<u32x2*>(kp + d * 2) = u32x2{T::pack(dk[mb][4 * i4] * fk, dk[mb][4 * i4 + 1] * fk), T::pack(dk[mb][4 * i4 + 2] * fk, dk[mb][4 * i4 + 3] * fk)};
      *reinterpret_cast<u32x2*>(vp + d * 2) = u32x2{T::pack(dv[mb][4 * i4] * fv, dv[mb][4 * i4 + 1] * fv), T::pack(dv[mb][4 * i4 + 2] * fv, dv[mb][4 * i4 + 3] * fv)};
    }
}

// adds the parts of split keys: items {-, -, k_start, k_len, first, first slot, slots, -}; a thread adds 4 channels of one key
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(const Params p) {
  const Item it = p.items[blockIdx.y / p.kv_heads];
  const int hk = blockIdx.y % p.kv_heads;
  const int at = blockIdx.x * 256 + threadIdx.x, row = at / (DP / 2), x = at % (DP / 2) * 4;         // x: dK's channels, then dV's
  const int key = it.first + row, d = x % DP;
  if (!item_ok(it, p) || key >= it.k_len || d >= p.dim || (long)it.begin + it.end > p.n_slots) return;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < it.end; ++i)
    sum += *reinterpret_cast<const f32x4*>(p.part + ((((long)(it.begin + i) * p.kv_heads + hk) * Dkv<DP>::KEYS) + row) * 2 * DP + x);
  const View& out = x < DP ? p.dk : p.dv;
  *reinterpret_cast<u32x2*>(const_cast<char*>(out.p) + (long)(it.k_start + key) * out.st + (long)hk * out.sh + d * 2) = u32x2{T::pack(sum.x, sum.y), T::pack(sum.z, sum.w)};
}

// ---------------------------------------------------------------------------------------------------------------- plan
constexpr long MAX_ROWS = 1l << 30;

int pad_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

bool heads_ok(int64_t heads, int64_t kv_heads, int64_t dim) {
  return kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads / kv_heads <= 32 && heads <= 65535 && dim >= 8 && dim <= 128 && dim % 8 == 0;
}

struct Writer {                                  // counts always, writes where there is room
  Item* out; long cap, n;
  void put(const Item& it) { if (out && n < cap) out[n] = it; ++n; }
};

long cost(const Item& it) { return (long)it.end - it.begin; }
bool longer(const Item& a, const Item& b) {
  if (cost(a) != cost(b)) return cost(a) > cost(b);
  if (a.q_start != b.q_start) return a.q_start < b.q_start;
  if (a.first != b.first) return a.first < b.first;
  return a.begin < b.begin;
}

bool view_ok(const View& t, long tokens, long heads, int dim, bool keys = false) {
  // 16-byte loads; a tile's offsets (up to 128 tokens and the heads of a group) stay below 2^31
  if (keys && tokens > 1 && t.st < 2 * dim) return false;
  return t.p && ((unsigned long)t.p & 15) == 0 && t.st >= 0 && t.sh >= 0 && t.st % 16 == 0 && t.sh % 16 == 0 && t.st < (1l << 40) && t.sh < (1l << 40) &&
         128 * t.st + 32 * t.sh + dim * 2 < (1l << 31);
}

unsigned clear_blocks(long rows, long heads, int dim) { return (unsigned)std::min<long>(1024, (rows * heads * dim * 2 + CLEAR_BYTES - 1) / CLEAR_BYTES); }

template <typename T, int DP, int NW> int launch_fwd(const Params& p, unsigned more, hipStream_t st) {
  if (p.blocks + more == 0) return DH_OK;
  hipLaunchKernelGGL((attn_fwd_kernel<T, DP, NW>), dim3(p.blocks + more), dim3(NW * 64), 0, st, p);
  DH_LAUNCH_CHECK();
  return DH_OK;
}
template <typename T, int DP> int run_fwd(Params p, const dh_attn_info& info, const Item* items, hipStream_t st) {
  p.items = items;
  p.blocks = (int)(info.n_fwd * info.kv_heads);
  const unsigned more = clear_blocks(p.q_rows - p.clear_q, p.heads, p.dim);
  const int rc = info.waves == 1 ? launch_fwd<T, DP, 1>(p, more, st) : launch_fwd<T, DP, 4>(p, more, st);
  if (rc != DH_OK) return rc;
  if (info.n_join) {
    p.items = items + info.n_fwd;
    const int rows = (int)info.waves * 32;
    hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3(rows / 8, (unsigned)(info.n_join * info.kv_heads)), dim3(256), 0, st, p, rows);
    DH_LAUNCH_CHECK();
  }
  return DH_OK;
}
template <typename T, int DP> int run_bwd(Params p, const dh_attn_info& info, const Item* items, hipStream_t st) {
  p.items = items + info.n_fwd + info.n_join;
  p.n_slots = info.n_dq_slots;
  p.blocks = (int)(info.n_dq * info.kv_heads);
  unsigned more = clear_blocks(p.q_rows - p.clear_q, p.heads, p.dim);
  if (p.blocks + more) {
    hipLaunchKernelGGL((attn_dq_kernel<T, DP, 4>), dim3(p.blocks + more), dim3(256), 0, st, p);
    DH_LAUNCH_CHECK();
  }
  p.items += info.n_dq;
  if (info.n_dq_join) {
    hipLaunchKernelGGL((attn_dq_join_kernel<T, DP>), dim3(128 * DP / 4 / 256, (unsigned)(info.n_dq_join * info.kv_heads)), dim3(256), 0, st, p);
    DH_LAUNCH_CHECK();
  }
  p.items += info.n_dq_join;
  p.n_slots = info.n_dkv_slots;
  p.blocks = (int)(info.n_dkv * info.kv_heads);
  more = clear_blocks(p.k_rows - p.clear_k, p.kv_heads, p.dim);
  if (p.blocks + more) {
    DH_LDS_OPTIN((attn_dkv_kernel<T, DP>), Dkv<DP>::LDS);
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP>), dim3(p.blocks + more), dim3(Dkv<DP>::WAVES * 64), Dkv<DP>::LDS, st, p);
    DH_LAUNCH_CHECK();
  }
  p.items += info.n_dkv;
  if (info.n_dkv_join) {
    hipLaunchKernelGGL((attn_dkv_join_kernel<T, DP>), dim3(Dkv<DP>::KEYS * DP / 2 / 256, (unsigned)(info.n_dkv_join * info.kv_heads)), dim3(256), 0, st, p);
    DH_LAUNCH_CHECK();
  }
  return DH_OK;
}

constexpr long MAX_THREADS = 0xffffffffl;         // of one launch

bool info_ok(const dh_attn_info* i) {
  if (!i || !heads_ok(i->heads, i->kv_heads, i->head_dim) || i->causal_block < 0 || i->causal_block > MAX_ROWS || (i->waves != 1 && i->waves != 4)) return false;
  const int64_t threads[3] = {i->waves * 64, 256, (pad_dim((int)i->head_dim) == 128 ? Dkv<128>::WAVES : Dkv<64>::WAVES) * 64};
  const int64_t items[3] = {i->n_fwd, i->n_dq, i->n_dkv}, joins[3] = {i->n_join, i->n_dq_join, i->n_dkv_join}, slots[3] = {i->n_slots, i->n_dq_slots, i->n_dkv_slots};
  int64_t n = 0;
  for (int k = 0; k < 3; ++k) {
    if (items[k] < 0 || items[k] > INT_MAX / 8 || (items[k] * i->kv_heads + 1024) * threads[k] > MAX_THREADS || joins[k] < 0 || joins[k] * i->kv_heads > 65535 || slots[k] < 0 || slots[k] > items[k]) return false;
    n += items[k] + joins[k];
  }
  return i->ints == 8 * n && i->q_rows >= 0 && i->k_rows >= 0 && i->q_rows <= MAX_ROWS && i->k_rows <= MAX_ROWS;
}

}  // namespace

extern "C" int dh_attn_plan(const int64_t* q_len, const int64_t* k_len, const int64_t* k_start, int64_t n_seqs, int heads, int kv_heads, int head_dim,
                            int64_t causal_block, int32_t* plan, int64_t plan_ints, dh_attn_info* info) {
  if (!info || n_seqs < 0 || (n_seqs && (!q_len || !k_len)) || !heads_ok(heads, kv_heads, head_dim) || causal_block < 0 || plan_ints < 0) return DH_ERR_ARG;
  const int block = (int)std::min<int64_t>(causal_block, MAX_ROWS), group = heads / kv_heads;
  long q_rows = 0, k_rows = 0, k_at = 0, most = 0;
  for (int64_t i = 0; i < n_seqs; ++i) {
    if (q_len[i] < 0 || k_len[i] < 0 || q_len[i] > MAX_ROWS || k_len[i] > MAX_ROWS) return DH_ERR_ARG;
    const long ks = k_start ? k_start[i] : k_at;
    if (ks < 0 || ks > MAX_ROWS) return DH_ERR_ARG;
    q_rows += q_len[i];
    k_at += k_len[i];
    k_rows = std::max(k_rows, ks + (k_len[i] ? k_len[i] : 0));
    most = std::max<long>(most, q_len[i]);
    if (q_rows > MAX_ROWS || k_rows > MAX_ROWS || k_at > (1l << 40)) return DH_ERR_ARG;
  }
  // rows a workgroup, one choice for all sequences: one wave where a tile of 32 holds every row of the longest, else 128 (32 single queries of 16/2 heads: 82 us against
  // 109 with 128 rows; 768 queries of 8 heads over 23040 keys: 90 us against 59 with 128)
  const int waves = most * group <= 32 ? 1 : 4;
  const int tpt = waves * 32 / group, tpt_q = 128 / group;
  // Long walks over the keys become several work items (pieces of whole key tiles, joined afterwards) where they would outlast the rest:
  // the aim is an equal share of all key tiles for each of the workgroups that the chip holds at once.  A walk is only split if that saves
  // 24 tiles (some 20 us) of a workgroup's walk: a split row's sums go through memory once more, and the join is a launch of its own (packed clips,
  // 64 channels: 87 us with 8, 85 with 24).  The limit looks at each walk alone and is the same for every head_dim: on training clips (64 channels) walks of 36
  // tiles stay whole beside a mean of 15, with all 648 workgroups on the chip at once, so that it empties while the longest end.
  // Lone waves are split for any saving: long walks meet short ones there, and a join is needed anyway (32 queries over 1 .. 32400 keys: 82 us; 87 if it had to
  // save 4 tiles, 130 if 24).
  const int dp = pad_dim(head_dim);
  struct Share {
    long piece, save;
    long pieces(long nt) const { return nt > piece + piece / 8 + save ? (nt + piece - 1) / piece : 1; }
  };
  const int64_t* ql = q_len; const int64_t* kl = k_len;
  auto share_of = [&](int step, long places, long save) {      // walks of `step` tokens each; places: workgroups that LDS or registers leave room for
    auto each_walk = [&](auto&& f) {
      for (int64_t i = 0; i < n_seqs; ++i)
        for (long t = 0; t < ql[i]; t += step) f((keys_seen((int)std::min<long>(ql[i], t + step) - 1, (int)ql[i], (int)kl[i], block) + BN - 1) / BN);
    };
    long tiles = 0, walks = 0;
    each_walk([&](long nt) { tiles += nt * kv_heads; walks += kv_heads; });
    Share s{std::max<long>(4, (tiles + places - 1) / places), save};
    if (walks < places)                          // rounding up must not leave a few items for a second round
      for (;;) {
        long n = 0, longest = 0;
        each_walk([&](long nt) { n += s.pieces(nt) * kv_heads; longest = std::max(longest, nt); });
        if (n <= places || longest <= s.piece) break;
        s.piece += std::max<long>(1, s.piece / 16);
      }
    return s;
  };
  const Share share = share_of(tpt, 256 * (waves == 1 ? (dp == 128 ? 3 : 6) : dp == 128 ? 2 : 3), waves == 1 ? 0 : 24);
  const Share share_q = share_of(tpt_q, 256 * (dp == 128 ? 2 : 3), 24);      // dQ: the forward's walk, always in tiles of 128 rows
  // The same for the rows of dK and dV.  A split key tile costs a trip of its 32-bit sums through memory, so pieces are 24 tiles of 64 rows at
  // least.  One share a place where three workgroups fit a CU; four where one does (training window, 128 channels: 3.20, 3.09, 3.04 ms with two,
  // one, four shares of 256; packed clips, 64 channels: 124, 121 us with two, one share of 768).
  long row_tiles = 0;
  auto rows_of = [&](int64_t i, long x) -> long {              // the first token that sees key x
    return block ? std::min<long>(q_len[i], std::max<long>(0, x / block * block - (k_len[i] - q_len[i]))) : 0;
  };
  const bool wide = pad_dim(head_dim) == 128;
  const int dkv_keys = wide ? Dkv<128>::KEYS : Dkv<64>::KEYS, tpt_k = (wide ? Dkv<128>::ROWS : Dkv<64>::ROWS) / group;
  for (int64_t i = 0; i < n_seqs; ++i)
    for (long x = 0; x < k_len[i]; x += dkv_keys) row_tiles += (q_len[i] - rows_of(i, x) + tpt_k - 1) / tpt_k * (long)kv_heads;
  const long shares = wide ? 1024 : 768, piece_k = std::max<long>(24, (row_tiles + shares - 1) / shares);
  Item* base = reinterpret_cast<Item*>(plan);
  const long cap = plan ? plan_ints / 8 : 0;
  Writer w{base, cap, 0};
  int64_t counts[6], slots[6];
  for (int pass = 0; pass < 6; ++pass) {         // forward items and joins, dQ items and joins, dK / dV items and joins
    const long from = w.n;
    long qs = 0, ka = 0, slot = 0;
    // a walk of nt tiles in n pieces: an item each (piece x: from tile a on, to tile b), or what joins them
    auto put = [&](Item it, long nt, long n, auto&& range) {
      if (pass % 2 == 0) {
        if (n == 1) w.put(it);
        else
          for (long x = 0; x < n; ++x) {
            range(it, nt * x / n, nt * (x + 1) / n);
            it.slot = (int)slot++;
            w.put(it);
          }
      } else if (n > 1) {
        it.begin = (int)slot;
        it.end = (int)n;
        slot += n;
        w.put(it);
      }
    };
    for (int64_t i = 0; i < n_seqs; ++i) {
      const int m = (int)q_len[i], n = (int)k_len[i];
      const int ks = (int)(k_start ? k_start[i] : ka);
      if (pass < 4) {
        const int step = pass < 2 ? tpt : tpt_q;
        for (int t = 0; t < m; t += step) {
          const int e = keys_seen(std::min(m, t + step) - 1, m, n, block);
          const long nt = (e + BN - 1) / BN;
          put(Item{(int)qs, m, ks, n, t, 0, e, -1}, nt, (pass < 2 ? share : share_q).pieces(nt), [&](Item& it, long a, long b) {
            it.begin = (int)(a * BN);
            it.end = (int)std::min<long>(e, b * BN);
          });
        }
      } else {
        for (int x = 0; x < n; x += dkv_keys) {
          const int t0 = (int)rows_of(i, x);
          const long nt = ((long)m - t0 + tpt_k - 1) / tpt_k;
          put(Item{(int)qs, m, ks, n, x, t0, m, -1}, nt, nt > piece_k + piece_k / 4 ? (nt + piece_k - 1) / piece_k : 1, [&](Item& it, long a, long b) {
            it.begin = (int)(t0 + a * tpt_k);
            it.end = (int)std::min<long>(m, t0 + b * tpt_k);
          });
        }
      }
      qs += m;
      ka += n;
      if (slot > INT_MAX || w.n > INT_MAX / 8) return DH_ERR_ARG;
    }
    slots[pass] = slot;
    counts[pass] = w.n - from;
    // longest first, so that the last workgroups to start are short ones
    if (pass % 2 == 0 && base && w.n <= cap) std::sort(base + from, base + w.n, longer);
  }
  // key ranges of two sequences that share rows: fine to read, but their gradients would be written twice
  bool shared = false;
  if (k_start && n_seqs) {
    int64_t* order = (int64_t*)malloc(sizeof(int64_t) * n_seqs);
    if (!order) return DH_ERR_WORKSPACE;
    int64_t n = 0;
    for (int64_t i = 0; i < n_seqs; ++i)
      if (k_len[i]) order[n++] = i;
    std::sort(order, order + n, [&](int64_t a, int64_t b) { return k_start[a] < k_start[b]; });
    for (int64_t i = 1; i < n; ++i) shared |= k_start[order[i - 1]] + k_len[order[i - 1]] > k_start[order[i]];
    free(order);
  }
  memset(info, 0, sizeof *info);
  info->ints = w.n * 8;
  info->heads = heads; info->kv_heads = kv_heads; info->head_dim = head_dim; info->causal_block = block;
  info->waves = waves;
  info->n_fwd = counts[0]; info->n_join = counts[1]; info->n_dq = counts[2]; info->n_dq_join = counts[3]; info->n_dkv = counts[4];
  info->n_dkv_join = counts[5];
  info->n_slots = slots[0]; info->n_dq_slots = slots[2]; info->n_dkv_slots = slots[4]; info->q_rows = q_rows; info->k_rows = k_rows; info->keys_shared = shared; info->k_total = k_at;
  if (!info_ok(info)) return DH_ERR_ARG;
  if (plan && plan_ints < info->ints) return DH_ERR_WORKSPACE;
  return DH_OK;
}

extern "C" size_t dh_attn_fwd_workspace_bytes(const dh_attn_info* info) {
  if (!info_ok(info)) return 0;
  return (size_t)info->n_slots * info->kv_heads * (info->waves * 32) * (pad_dim((int)info->head_dim) + 2) * sizeof(float);
}

extern "C" int dh_attn_fwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                           void* o, int64_t o_st, int64_t o_sh, void* o_low, float* lse, const int32_t* plan, const dh_attn_info* info, int dtype, int64_t q_rows,
                           int64_t k_rows, float scale, int clear_rest, void* workspace, size_t workspace_bytes, dh_stream_t stream) {
  if (!info_ok(info) || (dtype != DH_F16 && dtype != DH_BF16) || q_rows < info->q_rows || k_rows < info->k_rows || q_rows > MAX_ROWS || k_rows > MAX_ROWS ||
      !(scale > 0.f) || !(scale < 1e30f)) return DH_ERR_ARG;
  if (info->n_fwd == 0 && !(clear_rest && q_rows)) return DH_OK;
  Params p;
  memset(&p, 0, sizeof p);
  p.q = {(const char*)q, q_st * 2, q_sh * 2}; p.k = {(const char*)k, k_st * 2, k_sh * 2}; p.v = {(const char*)v, v_st * 2, v_sh * 2}; p.o = {(const char*)o, o_st * 2, o_sh * 2};
  const int dim = (int)info->head_dim;
  if ((info->ints && !plan) || !lse || ((unsigned long)o_low & 15) || !view_ok(p.q, q_rows, info->heads, dim) || !view_ok(p.o, q_rows, info->heads, dim)) return DH_ERR_ARG;
  if (info->k_rows && (!view_ok(p.k, k_rows, info->kv_heads, dim, true) || !view_ok(p.v, k_rows, info->kv_heads, dim, true))) return DH_ERR_ARG;
  if (info->n_slots && (!workspace || ((unsigned long)workspace & 15) || workspace_bytes < dh_attn_fwd_workspace_bytes(info))) return DH_ERR_WORKSPACE;
  p.low = (char*)o_low; p.lse = lse; p.part = (float*)workspace; p.n_slots = info->n_slots;
  p.kv_heads = (int)info->kv_heads; p.heads = (int)info->heads; p.group = p.heads / p.kv_heads; p.dim = dim; p.block = (int)info->causal_block;
  p.q_rows = (int)q_rows; p.k_rows = (int)k_rows; p.plan_q_rows = (int)info->q_rows; p.plan_k_rows = (int)info->k_rows; p.clear_q = clear_rest ? (int)info->q_rows : p.q_rows; p.clear_k = clear_rest ? (int)info->k_rows : p.k_rows; p.scale = scale; p.c = scale * LOG2E;
  const Item* items = reinterpret_cast<const Item*>(plan);
  hipStream_t st = (hipStream_t)stream;
  const int dp = pad_dim(dim);
  if (dtype == DH_F16) return dp == 32 ? run_fwd<F16, 32>(p, *info, items, st) : dp == 64 ? run_fwd<F16, 64>(p, *info, items, st) : run_fwd<F16, 128>(p, *info, items, st);
  return dp == 32 ? run_fwd<BF16, 32>(p, *info, items, st) : dp == 64 ? run_fwd<BF16, 64>(p, *info, items, st) : run_fwd<BF16, 128>(p, *info, items, st);
}

static size_t row_floats(const dh_attn_info* i) { return ((size_t)i->q_rows * i->heads * 3 + 3) / 4 * 4; }
extern "C" size_t dh_attn_bwd_workspace_bytes(const dh_attn_info* info) {
  if (!info_ok(info)) return 0;
  // the parts of dQ are joined before those of dK and dV are written
  const size_t dp = pad_dim((int)info->head_dim), keys = dp == 128 ? Dkv<128>::KEYS : Dkv<64>::KEYS;
  return (row_floats(info) + std::max((size_t)info->n_dq_slots * 128 * (dp + 1), (size_t)info->n_dkv_slots * keys * 2 * dp) * info->kv_heads) * sizeof(float);
}

extern "C" int dh_attn_bwd(const void* grad, int64_t g_st, int64_t g_sh, const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                           const void* v, int64_t v_st, int64_t v_sh, const void* o, int64_t o_st, int64_t o_sh, const void* o_low, const float* lse, void* dq, int64_t dq_st,
                           int64_t dq_sh, void* dk, int64_t dk_st, int64_t dk_sh, void* dv, int64_t dv_st, int64_t dv_sh, const int32_t* plan,
                           const dh_attn_info* info, int dtype, int64_t q_rows, int64_t k_rows, float scale, int clear_rest, void* workspace,
                           size_t workspace_bytes, dh_stream_t stream) {
  if (!info_ok(info) || info->keys_shared || (dtype != DH_F16 && dtype != DH_BF16) || q_rows < info->q_rows || k_rows < info->k_rows || q_rows > MAX_ROWS ||
      k_rows > MAX_ROWS || !(scale > 0.f) || !(scale < 1e30f)) return DH_ERR_ARG;
  const bool rest_q = clear_rest && q_rows > info->q_rows, rest_k = clear_rest && k_rows > info->k_rows;
  if (info->n_dq == 0 && info->n_dkv == 0 && !rest_q && !rest_k) return DH_OK;
  Params p;
  memset(&p, 0, sizeof p);
  p.q = {(const char*)q, q_st * 2, q_sh * 2}; p.k = {(const char*)k, k_st * 2, k_sh * 2}; p.v = {(const char*)v, v_st * 2, v_sh * 2}; p.o = {(const char*)o, o_st * 2, o_sh * 2};
  p.g = {(const char*)grad, g_st * 2, g_sh * 2}; p.dq = {(const char*)dq, dq_st * 2, dq_sh * 2}; p.dk = {(const char*)dk, dk_st * 2, dk_sh * 2}; p.dv = {(const char*)dv, dv_st * 2, dv_sh * 2};
  const int dim = (int)info->head_dim;
  if (info->ints && !plan) return DH_ERR_ARG;
  if (info->n_dq) {
    if (!lse || ((unsigned long)o_low & 15) || !view_ok(p.q, q_rows, info->heads, dim) || !view_ok(p.o, q_rows, info->heads, dim) || !view_ok(p.g, q_rows, info->heads, dim) ||
        !view_ok(p.dq, q_rows, info->heads, dim)) return DH_ERR_ARG;
    if (!workspace || ((unsigned long)workspace & 15) || workspace_bytes < dh_attn_bwd_workspace_bytes(info)) return DH_ERR_WORKSPACE;
  }
  if (rest_q && !view_ok(p.dq, q_rows, info->heads, dim)) return DH_ERR_ARG;
  if (rest_k && (!view_ok(p.dk, k_rows, info->kv_heads, dim) || !view_ok(p.dv, k_rows, info->kv_heads, dim))) return DH_ERR_ARG;
  if (info->n_dkv && (!view_ok(p.k, k_rows, info->kv_heads, dim, true) || !view_ok(p.v, k_rows, info->kv_heads, dim, true) || !view_ok(p.dk, k_rows, info->kv_heads, dim) ||
                      !view_ok(p.dv, k_rows, info->kv_heads, dim))) return DH_ERR_ARG;
  p.low = (char*)const_cast<void*>(o_low); p.lse = const_cast<float*>(lse); p.delta = (float*)workspace; p.row_values = info->q_rows * info->heads; p.part = (float*)workspace + row_floats(info);
  p.kv_heads = (int)info->kv_heads; p.heads = (int)info->heads; p.group = p.heads / p.kv_heads; p.dim = dim; p.block = (int)info->causal_block;
  p.q_rows = (int)q_rows; p.k_rows = (int)k_rows; p.plan_q_rows = (int)info->q_rows; p.plan_k_rows = (int)info->k_rows; p.clear_q = clear_rest ? (int)info->q_rows : p.q_rows; p.clear_k = clear_rest ? (int)info->k_rows : p.k_rows; p.scale = scale; p.c = scale * LOG2E;
  const Item* items = reinterpret_cast<const Item*>(plan);
  hipStream_t st = (hipStream_t)stream;
  const int dp = pad_dim(dim);
  if (dtype == DH_F16) return dp == 32 ? run_bwd<F16, 32>(p, *info, items, st) : dp == 64 ? run_bwd<F16, 64>(p, *info, items, st) : run_bwd<F16, 128>(p, *info, items, st);
  return dp == 32 ? run_bwd<BF16, 32>(p, *info, items, st) : dp == 64 ? run_bwd<BF16, 64>(p, *info, items, st) : run_bwd<BF16, 128>(p, *info, items, st);
}
