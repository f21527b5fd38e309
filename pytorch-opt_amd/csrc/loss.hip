// Losses of a language model's head on gfx950, from hidden states H [rows, d]
// and the head's weight W [vocab, d], without the caller holding the logits.
//
// With z = H·Wᵀ/T (T = 1 but for distillation), lse_r = log Σ_v exp z_rv and
// p = exp(z − lse), a row's loss and the slope of its logits H·Wᵀ are
//   cross entropy, target y, smoothing ε, penalty ζ:
//     lse − (1−ε)·z_y − (ε/V)·Σ_v z_v + ζ·lse²,
//     p·(1 + 2ζ·lse) − (1−ε)·[v = y] − ε/V;
//   distillation, a teacher's k logits t at ids v_k, q = softmax(t/T):
//     T²·(lse − Σ_k q_k·z_{v_k} + Σ_k q_k·log q_k),   T·(p − Σ_k q_k·[v = v_k]),
// so both are a dense p and a few sparse targets per row, and share the code:
//   S = a·(f·p − u − Σ_k q_k·[v = v_k]),  a = g_r·λ/T, f = 1 + 2ζ·lse, u = ε/V,
// g_r the gradient of the row's loss and λ = T². The gradients are
//   dH = S·W,   dW = Sᵀ·H.
//
// Rows without a target are left out (not multiplied by zero): a prologue
// lists the rows that count, and everything after it works on that list, whose
// length only the device knows. Then, for chunks of rows:
//   gather   the chunk's rows of H, padded, and zero rows of dH for left-out ones;
//   logits   one MFMA product, whose epilogue takes the maximum and the sum of
//            exponentials of each row's 64 columns and the targets' logits, and
//            for gradients keeps the block's logits in the workspace;
//   finish   joins a row's blocks to its normaliser, gives its loss and turns
//            the kept logits into S;
//   dH, dW   two MFMA products (dW summed over the chunks in fp32).
// A pass over V·rows logits is 2·rows·d·V operations, the three products
// 6·rows·d·V: gradients found in the forward call need no second pass over the
// logits (8·rows·d·V). bf16 runs on its own matrix instructions, fp32 on those
// of fp16 (two planes per operand, three products; 2.9 times fp32's rate), and
// where the rows are few on its own (few_rows). Where the rows' gradients come later (losses per row),
// the normaliser and the targets' logits are kept and the backward call forms S
// in the logits' epilogue.
//
// A target's logit is the one that entered the sum of exponentials, so that
// what it is off by cancels in lse − z_y and p − 1 where p is near 1 (with a
// separate dot product a loss of 0.1 was off by 1e-5). For the same reason lse
// is kept as the largest logit m and s = Σ exp(z − m): p = exp(z − m)/s.
#include <algorithm>
#include <cmath>

#include "aux_kernels.h"
#include "gemm_nt.h"
#include "split.h"

namespace pto {
namespace {

constexpr int kCols = 64;      // columns of a row that one entry of the statistics covers
constexpr int kMaxTeach = 1024;  // sparse targets per row
constexpr int64_t kMaxMarked = 393216;  // tokens whose marks (10 bytes per 64) fit in 64 KB of LDS
constexpr int64_t kChunkBytes = int64_t(2) << 30;  // kept logits of a chunk of rows
constexpr double kLn2 = 0.6931471805599453;

// bf16 inputs: a kept logit is how far it lies below its block's maximum, in
// log2, as a 16-bit fraction of 128 from the top. p is then off by at most
// 6.8e-4 (bf16's rounding of S: up to 3.9e-3) in the bytes that S takes in the
// end, and 0 stands for exponentials 2^-128 times the block's largest and
// less, which fp32 does not hold as normal numbers either. fp32 inputs keep
// fp32.
constexpr float kOctaves = 128.f;
constexpr float kNear = 0x1p-32f;  // least sum of exponentials of a row against a shared reference

// Sparse targets. Cross entropy has one per row, by listed row: the token, or
// -2 where it is outside the vocabulary, with the same share in every row.
// Distillation has k per row of the call, in the caller's order: the token, -1
// where there is none, -2 outside the vocabulary; q its share; put what of S to
// take off at the token (the first of equal ids has their sum, the others -1:
// nothing to do); entropy Σ q·log q.
struct Targets {
  int* one;
  float share;
  int* id;
  float *q, *put, *entropy;
  int* kept;   // per row: whether the row counts
  // a chunk's tokens as a bit set, by 64 columns and row ([blocks][cap]), with
  // the number of bits in the row before them, and the rank of each entry's
  // token in its row ([cap][k])
  unsigned long long* bits;
  uint16_t* before;
  uint16_t* rank;
};
// The targets of one row.
struct RowTargets {
  const Targets& t;
  int64_t at, row;
  int k;
  __device__ __forceinline__ int id(int e) const { return t.one ? t.one[at] : t.id[row * k + e]; }
  __device__ __forceinline__ float q(int e) const { return t.one ? t.share : t.q[row * k + e]; }
  __device__ __forceinline__ float put(int e) const { return t.one ? t.share : t.put[row * k + e]; }
  __device__ __forceinline__ float entropy() const { return t.one ? 0.f : t.entropy[row]; }
};

__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The teacher's softmax over a row's entries that are there (id >= 0, logit
// above -inf), one wave per row, its entries in registers (8192 x 64: 15 us).
__global__ void __launch_bounds__(256) kd_targets_kernel(const float* __restrict__ logit,
                                                         const int64_t* __restrict__ index, int64_t rows, int k,
                                                         int64_t vocab, float inv_temp, Targets t) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const float* lr = logit + r * k;
  const int64_t* ir = index + r * k;
  constexpr int PER = kMaxTeach / 64;
  float v[PER];
  unsigned there = 0;
  float m = -INFINITY;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = q * 64 + lane;
    v[q] = -INFINITY;
    if (e >= k) continue;
    v[q] = lr[e] * inv_temp;
    const int64_t id = ir[e];
    if (id >= 0 && !(v[q] == -INFINITY)) there |= 1u << q;
    t.id[r * k + e] = !(there >> q & 1) ? -1 : id < vocab ? (int)id : -2;
    if (there >> q & 1) m = fmaxf(m, v[q]);
  }
  m = wave_max(m);
  float s = 0.f;
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (there >> q & 1) s += expf(v[q] - m);
  const float logs = logf(wave_sum(s));
  float ent = 0.f;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = q * 64 + lane;
    const float logq = v[q] - m - logs, share = there >> q & 1 ? expf(logq) : 0.f;
    if (share != 0.f) ent += share * logq;
    if (e < k) t.q[r * k + e] = share;
  }
  ent = wave_sum(ent);
  const int any = __any(there != 0);
  if (lane == 0) {
    t.kept[r] = any;
    t.entropy[r] = ent;
  }
}

// list = the rows that count in order, then the others; count = how many
// count; losses 0. y: cross entropy's targets (listed to t.one as well), else
// t.kept says which rows count. weights: alpha = scale times the largest
// magnitude of those that count (for 16-bit S under rows' gradients: the rows
// are scaled by a common value in fp32, so that equal gradients cost no
// rounding); else scale, over the count for the mean. One workgroup of 16
// waves, each a run of rows, 64 at a time: the order is by row, and it is a
// chain of loads either way (8192 rows 10 us, 256 5).
__global__ void __launch_bounds__(1024) list_rows_kernel(const int64_t* __restrict__ y, int64_t ignore, int64_t vocab,
                                                         Targets t, int64_t rows, int* __restrict__ list,
                                                         int* __restrict__ count, float* __restrict__ losses,
                                                         const float* __restrict__ weights, float scale, int mean,
                                                         float* __restrict__ alpha) {
  __shared__ int part[16];
  __shared__ float big[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t per = (rows + 1023) / 1024 * 64, r0 = w * per, r1 = min(rows, r0 + per);
  auto counts = [&](int64_t r) { return r < r1 && (y ? y[r] != ignore : t.kept[r] != 0); };
  int n = 0;
  float m = 0.f;
  // eight loads in flight
  for (int64_t b = r0; b < r0 + per; b += 512) {
    bool c[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) c[q] = counts(b + 64 * q + lane);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int64_t r = b + 64 * q + lane;
      n += __popcll(__ballot(c[q]));
      if (weights && c[q] && fabsf(weights[r]) < INFINITY) m = fmaxf(m, fabsf(weights[r]));
      if (losses && r < r1) losses[r] = 0.f;
    }
  }
  m = wave_max(m);
  if (lane == 0) {
    part[w] = n;
    big[w] = m;
  }
  __syncthreads();
  int yes = 0, total = 0;
  for (int o = 0; o < 16; ++o) {
    if (o < w) yes += part[o];
    total += part[o];
    m = fmaxf(m, big[o]);
  }
  int64_t no = total + min(rows, r0) - yes;
  for (int64_t b = r0; b < r0 + per; b += 512) {
    bool c[8];
    int64_t id[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int64_t r = b + 64 * q + lane;
      c[q] = counts(r);
      id[q] = y && r < r1 ? y[r] : 0;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int64_t r = b + 64 * q + lane;
      const unsigned long long mask = __ballot(c[q]);
      const int at = __popcll(mask & ((1ull << lane) - 1)), here = __popcll(mask);
      if (c[q]) {
        list[yes + at] = (int)r;
        if (y) t.one[yes + at] = id[q] >= 0 && id[q] < vocab ? (int)id[q] : -2;
      } else if (r < r1) {
        list[no + lane - at] = (int)r;
      }
      yes += here;
      no += 64 - here;
    }
  }
  if (threadIdx.x == 0) {
    count[0] = total;
    alpha[0] = weights ? (m > 0.f ? scale * m : scale) : mean ? scale / (float)max(total, 1) : scale;
  }
}

// What the products read: bf16, fp32 as two fp16 planes (sp16), or, for few
// rows, fp32 itself.
template <class O>
constexpr bool kPlanes = std::is_same<O, sp16>::value;
template <class O>
using Elem = std::conditional_t<kPlanes<O>, float, O>;

// The rows of a chunk, as the kernels see them.
struct Chunk {
  const int* list;
  const int* count;
  int64_t rows;  // of the call
  int base, cap;  // first listed row, most rows
  // count null: all of them
  __device__ __forceinline__ int live() const { return count ? max(0, min(cap, count[0] - base)) : cap; }
  // rows that products reading them along K see: zero rows up to a multiple of kPadK
  __device__ __forceinline__ int padded() const { return (live() + kPadK - 1) / kPadK * kPadK; }
};

// Distillation: the bit sets, ranks and shares by token of a chunk's rows,
// `several` (a power of two) a workgroup: the bit sets lie by block and row, and
// single words scattered over them took 87 us of 8192 rows' 64 targets among
// 32000, lines of eight rows 34. LDS: 10 bytes per 64 tokens and row.
__global__ void __launch_bounds__(256) mark_targets_kernel(Chunk ch, int blocks, int several, int k, Targets t) {
  extern __shared__ unsigned long long words[];
  uint16_t* const befores = reinterpret_cast<uint16_t*>(words + (int64_t)several * blocks);
  __shared__ int part[256];
  __shared__ int entries[8];
  const int tid = threadIdx.x, each = 256 / several, r = tid / each, of = tid % each;
  const int i = blockIdx.x * several + r, live = ch.live();
  if ((int)blockIdx.x * several >= live) return;
  const int64_t row = i < live ? ch.list[ch.base + i] : 0;
  const int* id = t.id + row * k;
  unsigned long long* const word = words + (int64_t)r * blocks;
  uint16_t* const before = befores + (int64_t)r * blocks;
  for (int b = of; b < blocks; b += each) word[b] = 0;
  if (of == 0) entries[r] = 0;
  __syncthreads();
  if (i < live)
    for (int e = of; e < k; e += each) {
      const int v = id[e];
      if (v < 0) continue;
      atomicOr(&word[v >> 6], 1ull << (v & 63));
      atomicAdd(&entries[r], 1);
    }
  __syncthreads();
  const int per = (blocks + each - 1) / each, b0 = min(blocks, of * per), b1 = min(blocks, b0 + per);
  int n = 0;
  for (int b = b0; b < b1; ++b) n += __popcll(word[b]);
  part[tid] = n;
  __syncthreads();
  for (int o = 1; o < each; o <<= 1) {
    const int add = of >= o ? part[tid - o] : 0;
    __syncthreads();
    part[tid] += add;
    __syncthreads();
  }
  int run = part[tid] - n;
  for (int b = b0; b < b1; ++b) {
    before[b] = (uint16_t)run;
    run += __popcll(word[b]);
  }
  __syncthreads();
  if (t.bits)
    for (int q = tid; q < blocks * several; q += 256) {
      const int b = q / several, at = blockIdx.x * several + q % several;
      if (at >= ch.cap) continue;
      t.bits[(int64_t)b * ch.cap + at] = words[(int64_t)(q % several) * blocks + b];
      t.before[(int64_t)b * ch.cap + at] = befores[(int64_t)(q % several) * blocks + b];
    }
  if (i >= live) return;
  const bool repeats = part[r * each + each - 1] != entries[r];
  for (int e = of; e < k; e += each) {
    const int v = id[e];
    float put = -1.f;
    if (v >= 0) {
      t.rank[(int64_t)i * k + e] = (uint16_t)(before[v >> 6] + __popcll(word[v >> 6] & ((1ull << (v & 63)) - 1)));
      put = t.q[row * k + e];
      if (repeats) {
        put = 0.f;
        for (int o = 0; o < k; ++o) {
          if (id[o] != v) continue;
          if (o < e) {
            put = -1.f;
            break;
          }
          put += t.q[row * k + o];
        }
      }
    }
    t.put[row * k + e] = put;
  }
}

// A row of n elements (any alignment) into a padded one, one wave.
template <typename T>
__device__ __forceinline__ void copy_row(const T* __restrict__ src, int64_t n, T* __restrict__ dst, int64_t ld,
                                         int lane) {
  constexpr int E = 16 / (int)sizeof(T), STEP = 64 * E;
  int64_t c = lane * E;
  for (; c + 3 * STEP + E <= n; c += 4 * STEP) {  // loads in flight
    uint4 u[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) u[q] = ld16(src + c + q * STEP);
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(dst + c + q * STEP) = u[q];
  }
  for (; c < ld; c += STEP) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (c + E <= n) {
      u = ld16(src + c);
    } else if (c < n) {
      T* e = reinterpret_cast<T*>(&u);
      for (int k = 0; k < E; ++k)
        if (c + k < n) e[k] = src[c + k];
    }
    *reinterpret_cast<uint4*>(dst + c) = u;
  }
}

// The chunk's rows of H together, at the copy's rate (8192 x 2048: 15 us), and
// dH of left-out rows.
template <typename T>
__device__ __forceinline__ void zero_row(T* __restrict__ row, int64_t d, int lane) {
  for (int64_t c = lane; c < d; c += 64) row[c] = T(0.f);
}
template <typename T>
__global__ void __launch_bounds__(256) gather_kernel(Chunk ch, const T* __restrict__ h, int64_t ldh, int64_t d,
                                                     T* __restrict__ hc, int64_t ldc, T* __restrict__ dh) {
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i < ch.live())
    copy_row(h + ch.list[ch.base + i] * ldh, d, hc + i * ldc, ldc, lane);
  else if (i < ch.padded())
    copy_row(h, 0, hc + i * ldc, ldc, lane);
  if (dh && i >= ch.live() && i < ch.cap) zero_row(dh + ch.list[ch.base + i] * d, d, lane);
}

// W padded to a multiple of kPadK rows and columns (50001 x 1000: 32 us).
template <typename T>
__global__ void __launch_bounds__(256) pad_weight_kernel(const T* __restrict__ w, int64_t ldw, int64_t vocab,
                                                         int64_t d, T* __restrict__ out, int64_t ldo, int64_t rows) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  copy_row(w + min(r, vocab - 1) * ldw, r < vocab ? d : 0, out + r * ldo, ldo, threadIdx.x & 63);
}

// The rows of W from the last multiple of kPadK on, at W's pitch and with zero
// rows up to the next (tail), and its last row by itself, padded to ldo.
template <typename T>
__global__ void __launch_bounds__(256) weight_tail_kernel(const T* __restrict__ w, int64_t ldw, int64_t vocab,
                                                          int64_t d, T* __restrict__ tail, T* __restrict__ last,
                                                          int64_t ldo) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t v = vocab / kPadK * kPadK + r;
  if (tail) copy_row(w + min(v, vocab - 1) * ldw, v < vocab ? d : 0, tail + r * ldw, ldw, lane);
  if (last && r == 0) copy_row(w + (vocab - 1) * ldw, d, last, ldo, lane);
}

// Four values of a row of n (the rest 0).
__device__ __forceinline__ void load_columns(const float* p, int n, float (&v)[4]) {
  uint4 u = make_uint4(0, 0, 0, 0);
  if (n >= 4) {
    u = ld16(p);
  } else {
    if (n > 0) u.x = __float_as_uint(p[0]);
    if (n > 1) u.y = __float_as_uint(p[1]);
    if (n > 2) u.z = __float_as_uint(p[2]);
  }
  v[0] = __uint_as_float(u.x);
  v[1] = __uint_as_float(u.y);
  v[2] = __uint_as_float(u.z);
  v[3] = __uint_as_float(u.w);
}
// A row of n floats as split planes (padded to ld, pl elements apart) with the
// exponent of its largest finite value, one wave; copy: also as it is. The
// second reading comes from cache (W of 32001 x 1024: 62 us, 4.2 TB/s).
__device__ __forceinline__ void row_planes(const float* __restrict__ src, int64_t n, sp16* __restrict__ dst, int64_t pl,
                                           int64_t ld, int* __restrict__ exponent, float* __restrict__ copy, int lane) {
  float m = 0.f;
#pragma unroll 4
  for (int64_t c = lane * 4; c < n; c += 256) {
    float v[4];
    load_columns(src + c, (int)(n - c), v);
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fabsf(v[k]) < INFINITY ? fmaxf(m, fabsf(v[k])) : m;
  }
  const int e = split_exp(wave_max(m));
  if (lane == 0) *exponent = e;
  for (int64_t c = lane * 8; c < ld; c += 512) {
    float lo[4], hi[4], v[8];
    load_columns(src + c, (int)(n - c), lo);
    load_columns(src + c + 4, (int)(n - c) - 4, hi);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < 4 ? lo[k & 3] : hi[k & 3];
    if (copy) st8<float, float>(copy + c, v, 0, 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], e);
    const Split8 s = split8(v);
    *reinterpret_cast<uint4*>(dst + c) = s.h;
    *reinterpret_cast<uint4*>(dst + pl + c) = s.l;
  }
}
__global__ void __launch_bounds__(256) weight_planes_kernel(const float* __restrict__ w, int64_t ldw, int64_t vocab,
                                                            int64_t d, sp16* __restrict__ out, int64_t ld,
                                                            int* __restrict__ exponent) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r < vocab) row_planes(w + r * ldw, d, out + r * ld, vocab * ld, ld, exponent + r, nullptr, threadIdx.x & 63);
}
// gather_kernel for planes: H as it is and as planes; also clears the maxima of
// the chunk's columns.
__global__ void __launch_bounds__(256) gather_planes_kernel(Chunk ch, const float* __restrict__ h, int64_t ldh,
                                                            int64_t d, float* __restrict__ hc, int64_t ldc,
                                                            sp16* __restrict__ planes, int64_t pl,
                                                            int* __restrict__ exponent, float* __restrict__ dh,
                                                            unsigned* __restrict__ maxima, int64_t nmax) {
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < nmax; c += (int64_t)gridDim.x * 256) maxima[c] = 0;
  if (i < ch.live())
    row_planes(h + ch.list[ch.base + i] * ldh, d, planes + i * ldc, pl, ldc, exponent + i, hc + i * ldc, lane);
  else if (i < ch.padded())
    copy_row(h, 0, hc + i * ldc, ldc, lane);
  if (dh && i >= ch.live() && i < ch.cap) zero_row(dh + ch.list[ch.base + i] * d, d, lane);
}

// 2^x of one v_exp_f32 (1 ulp; results below 2^-126 are 0).
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// ------------------------------------------------------------ the logits

// Exchange within 16 consecutive lanes (the lanes of one row of an
// accumulator): neighbours, pairs, halves, the rest.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp<0xB1>(v));      // quad_perm 1 0 3 2
  v = fmaxf(v, dpp<0x4E>(v));      // quad_perm 2 3 0 1
  v = fmaxf(v, dpp<0x141>(v));     // row_half_mirror
  return fmaxf(v, dpp<0x140>(v));  // row_mirror
}
__device__ __forceinline__ float sum16(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  return v + dpp<0x140>(v);
}

// Sums of four values over 16 lanes each: lane l gets the sum of v[l & 3].
__device__ __forceinline__ float sum_rows(const float (&v)[4], int l) {
  const bool odd = l & 1, up = l & 2;
  const float a = (odd ? v[1] : v[0]) + dpp<0xB1>(odd ? v[0] : v[1]);
  const float b = (odd ? v[3] : v[2]) + dpp<0xB1>(odd ? v[2] : v[3]);
  float s = (up ? b : a) + dpp<0x4E>(up ? a : b);
  s += dpp<0x124>(s);  // row_ror 4
  return s + dpp<0x128>(s);  // row_ror 8
}

// What a row's slopes need besides its logits t (in log2): S = pa·2^(t − m) + pu.
struct RowSlope {
  float m, pa, pu;
};

// Epilogue of the logits' product, from the accumulators (kDirect): 16 lanes
// have a row's 64 columns, four each. Through LDS staging in runs of eight the
// same work took 14 us of a 256² tile's 69 at d = 2048, most of it VALU. Now a
// round of tiles takes 47 us per 2048 of d and 8.5 besides (12 where logits are
// kept): 8192 x 2048 x 32000 1018 us, 1.05 PFLOP/s (dH and dW of that size 857).
// Split operands come with a power of two per row of each.
template <class O, bool KEEP, bool SLOPE>
struct EpiLogits {
  typedef Elem<O> T;
  typedef char S;  // the staging slice holds a row's targets and scales, no values
  static constexpr bool kDirect = true;
  Chunk ch;
  int vocab;
  float scale;     // log2(e)/T
  float2* stats;   // [cap][blocks]: maximum, Σ 2^(t − maximum)
  float* sums;     // [cap][blocks] or null: Σ t
  int64_t blocks;
  void* kept;      // KEEP: the kept logits (uint16_t or float); SLOPE: S
  int64_t ld;
  const RowSlope* row;
  const int *eh, *ew;  // planes: the exponents of the rows of H and W
  Targets tg;
  int k;
  float* targets;  // [cap][k], null: the targets' logits t, by rank
  bool in_place;   // P is H itself, its rows by the list
  const void* last;  // a padded copy of W's last row, where its rows are read past their ends
  __device__ __forceinline__ bool adjust(GemmArgs& g, int, int row0, int) const {
    g.M = SLOPE ? ch.padded() : ch.live();
    return row0 < g.M;
  }
  __device__ __forceinline__ int p_row(int i) const { return in_place ? ch.list[ch.base + i] : i; }
  __device__ __forceinline__ const void* q_last() const { return kPlanes<O> ? nullptr : last; }
  __device__ __forceinline__ int q_rows() const { return vocab; }
  __device__ __forceinline__ void finish(int) const {}
  template <class V, int FM, int FN>
  __device__ __forceinline__ void direct(const V (&acc)[FM][FN], char* lds, const GemmArgs& g, int wr0, int wc0,
                                         int lane) const {
    if (wc0 >= g.N || wr0 >= g.M) return;
    const int l = lane & 15, sub = (lane >> 4) * 4, c0 = wc0 + 4 * l;
    const bool whole = wc0 + kCols <= vocab;  // false in the last block of a row at most
    RowSlope* const rs = reinterpret_cast<RowSlope*>(lds);
    constexpr int R = FM * 16;
    unsigned long long* const bits = reinterpret_cast<unsigned long long*>(lds);
    uint16_t* const before = reinterpret_cast<uint16_t*>(bits + R);
    int* const er = reinterpret_cast<int*>(before + R);
    int ec[4] = {0, 0, 0, 0};
    // rows with a target in these columns, one bit each
    unsigned long long hit[(R + 63) / 64] = {};
    if (targets) {
#pragma unroll
      for (int q = 0; q < (R + 63) / 64; ++q) {
        const int r = q * 64 + lane, i = wr0 + r;
        unsigned long long word = 0;
        int first = 0;
        if (r < R && i < g.M) {
          if (tg.one) {
            const unsigned at = (unsigned)tg.one[ch.base + i] - wc0;  // -2: past every block
            word = at < kCols ? 1ull << at : 0;
          } else {
            const int64_t at = (int64_t)(wc0 / kCols) * ch.cap + i;
            word = tg.bits[at];
            first = tg.before[at];
          }
        }
        hit[q] = __ballot(word != 0);
        if (r < R) {
          bits[r] = word;
          before[r] = (uint16_t)first;
        }
      }
    }
    if (kPlanes<O>) {
      for (int r = lane; r < R; r += 64) er[r] = eh[min(wr0 + r, g.M - 1)];
#pragma unroll
      for (int k = 0; k < 4; ++k) ec[k] = ew[min(c0 + k, vocab - 1)];
    }
    if (SLOPE) {
      for (int r = lane; r < R; r += 64)
        if (wr0 + r < g.M) rs[r] = row[wr0 + r];
    }
    __builtin_amdgcn_s_waitcnt(PTO_LGKM0);
    __builtin_amdgcn_wave_barrier();
    auto value = [&](int fm, int r, int k) {
      const float v = acc[fm][k][r];
      return kPlanes<O> ? ldexpf(v, -er[fm * 16 + sub + r] - ec[k]) : v;
    };
    if (targets) {
#pragma unroll
      for (int fm = 0; fm < FM; ++fm) {
        if (((hit[fm / 4] >> (fm % 4 * 16)) & 0xffff) == 0) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if ((hit[fm / 4] >> (fm % 4 * 16 + r) & 0x1111) == 0) continue;
          const int at = fm * 16 + sub + r;
          const unsigned long long word = bits[at];
          const int first = before[at];
          unsigned mine = (unsigned)(word >> (4 * l)) & 15u;
          if (mine == 0) continue;
          // most often one: a select and a store, not four of each
          float* to = targets + (int64_t)(wr0 + at) * k + first + __popcll(word & ((1ull << (4 * l)) - 1));
          const float v[4] = {value(fm, r, 0), value(fm, r, 1), value(fm, r, 2), value(fm, r, 3)};
          do {
            const unsigned c = __builtin_ctz(mine);
            *to++ = (c & 2 ? (c & 1 ? v[3] : v[2]) : (c & 1 ? v[1] : v[0])) * scale;
            mine &= mine - 1;
          } while (mine);
        }
      }
    }
    if constexpr (SLOPE) {
#pragma unroll
      for (int fm = 0; fm < FM; ++fm)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = wr0 + fm * 16 + sub + r;
          const RowSlope p = rs[fm * 16 + sub + r];
          float t[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            t[k] = fmaf(p.pa, pow2(fmaf(value(fm, r, k), scale, -p.m)), p.pu);
            if (!whole) t[k] = c0 + k < vocab ? t[k] : 0.f;
          }
          if (i < g.M)
            st4(reinterpret_cast<T*>(static_cast<char*>(kept) + ((int64_t)(wr0 + fm * 16 + r) * ld + wc0) * (int64_t)sizeof(T) +
                                     (unsigned)(sub * ld + 4 * l) * (unsigned)sizeof(T)),
                t);
        }
      return;
    }
    // One reference for all of the wave's values: 0 or the largest. Kept logits
    // and exponentials have the same relative precision however far below it
    // they lie, so it serves every row whose own maximum is at most 2^kNear
    // below; then a maximum per row (8 lane exchanges for each, half the
    // epilogue's instructions) is not needed.
    if (whole && wr0 + R <= g.M) {
      // uniform row addresses and a 32-bit offset per lane: 64-bit products per
      // lane and row cost 2 us a tile
      char* const krow = static_cast<char*>(kept) + ((int64_t)wr0 * ld + wc0) * (int64_t)sizeof(T);
      const unsigned klane = (unsigned)(sub * ld + 4 * l) * (unsigned)sizeof(T);
      char* const srow = reinterpret_cast<char*>(stats + (int64_t)wr0 * blocks + wc0 / kCols);
      const unsigned slane = (unsigned)((sub + (l & 3)) * blocks) * 8u;
      const bool mine = (l & 12) == 0;
      // the order of non-negative floats is that of their bits; what is not a
      // number is above them all
      int top = 0;
#pragma unroll
      for (int fm = 0; fm < FM; ++fm)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, __float_as_int(value(fm, r, k)));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
      const float ref = __int_as_float(__builtin_amdgcn_readfirstlane(top)) * scale;
      float least = INFINITY;
      if (ref < INFINITY) {
#pragma unroll
        for (int fm = 0; fm < FM; ++fm) {
          float s[4], z[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = value(fm, r, k);
            s[r] = (pow2(fmaf(v[0], scale, -ref)) + pow2(fmaf(v[1], scale, -ref))) +
                   (pow2(fmaf(v[2], scale, -ref)) + pow2(fmaf(v[3], scale, -ref)));
            if (sums) z[r] = (v[0] + v[1]) + (v[2] + v[3]);
            if (KEEP) keep(krow + (int64_t)(fm * 16 + r) * ld * (int64_t)sizeof(T), klane, v, ref);
          }
          // lane l: the sum of row r = l & 3
          const float sum = sum_rows(s, l);
          least = fminf(least, sum);
          if (mine) *reinterpret_cast<float2*>(srow + (int64_t)(fm * 16) * blocks * 8 + slane) = make_float2(ref, sum);
          if (sums) {
            const float zs = sum_rows(z, l) * scale;
            if (mine) sums[(int64_t)(wr0 + fm * 16 + sub + (l & 3)) * blocks + wc0 / kCols] = zs;
          }
        }
        if (!__any(!(least >= kNear))) return;
      }
    }
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      if (wr0 + fm * 16 >= g.M) break;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wr0 + fm * 16 + sub + r;
        const bool live = i < g.M;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] = value(fm, r, k);
          if (!whole) v[k] = c0 + k < vocab ? v[k] : -INFINITY;
        }
        const float m = max16(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
        const float ref = m == -INFINITY ? 0.f : m * scale;  // a block of nothing but -inf sums to 0
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) s += pow2(fmaf(v[k], scale, -ref));
        s = sum16(s);
        if (live && l == 0) stats[i * blocks + wc0 / kCols] = make_float2(ref, s);
        if (sums) {
          float z = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) z += c0 + k < vocab ? v[k] : 0.f;
          z = sum16(z) * scale;
          if (live && l == 0) sums[i * blocks + wc0 / kCols] = z;
        }
        if (KEEP && live) keep(static_cast<char*>(kept) + ((int64_t)i * ld + c0) * (int64_t)sizeof(T), 0, v, ref);
      }
    }
  }
  // Four columns of a row, kept.
  __device__ __forceinline__ void keep(char* row, unsigned at, const float (&v)[4], float ref) const {
    if constexpr (sizeof(T) == 2) {
      // 1 + (t − ref)/128 of 65535, rounded, between 0 and 65535
      const float f = scale / kOctaves, o = fmaf(-ref, 1.f / kOctaves, 1.f);
      auto two = [&](float a, float b) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(fmaf(a, f, o), fmaf(b, f, o)));
      };
      *reinterpret_cast<uint2*>(row + at) = make_uint2(two(v[0], v[1]), two(v[2], v[3]));
    } else {
      *reinterpret_cast<float4*>(row + at) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
    }
  }
  template <typename U>
  __device__ __forceinline__ static void st4(U* p, const float (&t)[4]) {
    struct __attribute__((aligned(4 * sizeof(U)))) Run {
      U e[4];
    };
    Run u;
#pragma unroll
    for (int k = 0; k < 4; ++k) u.e[k] = convert<U>(t[k]);
    *reinterpret_cast<Run*>(p) = u;
  }
};

// ------------------------------------------------------------ rows

struct LossSpec {
  float lambda;   // T² (1 for cross entropy)
  float smooth;   // ε/V
  float zeta;
  int k;
};

// Where the logits overflow, or a target is outside the vocabulary or not a
// number, nothing of the row is left standing as a number.
__device__ __forceinline__ bool sound(float x) { return fabsf(x) < INFINITY; }

// A row of S, times a.
__device__ __forceinline__ RowSlope row_slope(const LossSpec& sp, float2 norm, float qz, float a) {
  const float lse2 = norm.x + log2f(norm.y);
  RowSlope r;
  r.m = norm.x;
  r.pa = sound(lse2) && sound(qz) ? a * (1.f + 2.f * sp.zeta * (float)(kLn2 * lse2)) / norm.y : NAN;
  r.pu = -a * sp.smooth;
  return r;
}
// S at a sparse target with logit z, S being scaled by a.
__device__ __forceinline__ float at_target(const RowSlope& rs, float a, float put, float z) {
  return fmaf(rs.pa, pow2(z - rs.m), fmaf(-a, put, rs.pu));
}
// Planes: S/a of a row, its a, and the largest |S/a| of every column, as bits.
struct RowsOut {
  RowSlope* slope;
  float* a;
  unsigned* maxima;
  __device__ __forceinline__ void put(int i, const LossSpec& sp, float2 norm, float qz, float av, const RowTargets& t,
                                      const float* z, int first, int step) const {
    const RowSlope rs = row_slope(sp, norm, qz, 1.f);
    if (first == 0) {
      slope[i] = rs;
      a[i] = av;
    }
    for (int e = first; e < t.k; e += step)
      if (t.id(e) >= 0 && t.put(e) >= 0.f) {
        const float v = fabsf(at_target(rs, 1.f, t.put(e), z[e]));
        if (v < INFINITY) atomicMax(&maxima[t.id(e)], __float_as_uint(v));
      }
  }
};

// Workgroups (y) per listed row, each with a run of its columns (few rows would
// leave CUs idle): the normaliser, the loss and, for gradients
// (SLOPES), S/alpha in place of the kept logits or what the passes over them
// need (planes). losses is per row of the call; norm (m, s) and z (the
// targets' logits in the caller's order) per listed row. Bound by the logits'
// way in and out: 8192 x 32000 bf16 211 us, 5.0 TB/s.
template <class O, bool SLOPES>
__global__ void __launch_bounds__(256) finish_kernel(Chunk ch, const float2* __restrict__ stats,
                                                     const float* __restrict__ sums, int64_t blocks, LossSpec sp,
                                                     Targets tg, const float* __restrict__ caught, int vocab,
                                                     Elem<O>* __restrict__ kept, int64_t ld, RowsOut out,
                                                     const float* __restrict__ alpha, float* __restrict__ losses,
                                                     float2* __restrict__ norms, float* __restrict__ z) {
  typedef Elem<O> T;
  constexpr int E = 16 / (int)sizeof(T);
  const int i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t c0 = ld / kCols * blockIdx.y / gridDim.y * kCols, c1 = ld / kCols * (blockIdx.y + 1) / gridDim.y * kCols;
  if (i >= ch.live()) {
    if (SLOPES && !kPlanes<O> && i < ch.padded())
      for (int64_t c = c0 + tid * E; c < c1; c += 256 * E) *reinterpret_cast<uint4*>(kept + i * ld + c) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int row = ch.list[ch.base + i];
  const float2* st = stats + i * blocks;
  const RowTargets rt{tg, ch.base + i, row, sp.k};
  float* zr = z + (int64_t)(ch.base + i) * sp.k;
  __shared__ float red[4][4];
  float m = -INFINITY;
  for (int64_t c = tid; c < blocks; c += 256)
    if (st[c].y != 0.f) m = fmaxf(m, st[c].x + log2f(st[c].y));
  m = wave_max(m);
  if (lane == 0) red[0][w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  if (m == -INFINITY) m = 0.f;
  // targets around m: what is summed is small where the row is right
  float s = 0.f, sz = 0.f, qz = 0.f;
  for (int64_t c = tid; c < blocks; c += 256) {
    s += st[c].y == 0.f ? 0.f : st[c].y * exp2f(st[c].x - m);
    if (sums) sz += sums[i * blocks + c] - m * (float)max((int64_t)0, min((int64_t)kCols, vocab - c * kCols));
  }
  for (int e = tid; e < sp.k; e += 256) {
    const int id = rt.id(e);
    float ze = 0.f;
    if (id != -1) {
      ze = id < 0 ? NAN : caught[tg.one ? i : (int64_t)i * sp.k + tg.rank[(int64_t)i * sp.k + e]];
      qz += rt.q(e) * (ze - m);
    }
    if (blockIdx.y == 0) zr[e] = ze;
  }
  s = wave_sum(s);
  sz = wave_sum(sz);
  qz = wave_sum(qz);
  if (lane == 0) {
    red[1][w] = s;
    red[2][w] = sz;
    red[3][w] = qz;
  }
  __syncthreads();
  s = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  sz = red[2][0] + red[2][1] + red[2][2] + red[2][3];
  qz = red[3][0] + red[3][1] + red[3][2] + red[3][3];
  const float2 norm = make_float2(m, s);
  if (tid == 0 && blockIdx.y == 0) {
    const double logs = log2((double)s);
    const double nat = kLn2 * (logs - ((double)qz + (double)sp.smooth * sz)) + rt.entropy();
    const double lse = kLn2 * ((double)m + logs);
    losses[row] = (float)(sp.lambda * nat + (double)sp.zeta * lse * lse);
    norms[ch.base + i] = norm;
  }
  if constexpr (SLOPES) {
    if constexpr (kPlanes<O>) {
      out.put(i, sp, norm, qz, alpha[0], rt, zr, tid, 256);
      return;
    }
    const RowSlope rs = row_slope(sp, norm, qz, 1.f);
    for (int64_t c = c0 + tid * E; c < c1; c += 256 * E) {
      const uint4 u = *reinterpret_cast<const uint4*>(kept + i * ld + c);
      const unsigned uw[4] = {u.x, u.y, u.z, u.w};
      const float off = (st[c / kCols].x - m) - kOctaves;
      float p[E], o[8];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (sizeof(T) == 4) {
          p[e] = pow2(__uint_as_float(uw[e]) - m);
        } else {
          const unsigned x = e & 1 ? uw[e / 2] >> 16 : uw[e / 2] & 0xffffu;
          p[e] = x ? pow2(fmaf((float)x, kOctaves / 65535.f, off)) : 0.f;
        }
        o[e] = c + e < vocab ? fmaf(rs.pa, p[e], rs.pu) : 0.f;
      }
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(kept + i * ld + c) = make_float4(o[0], o[1], o[2], o[3]);
      else
        st8<bf16, float>(kept + i * ld + c, o, 0, 8);
    }
    __syncthreads();  // the dense part is written before the targets' entries replace theirs
    for (int e = tid; e < sp.k; e += 256) {
      const int id = rt.id(e);
      if (id >= c0 && id < c1 && rt.put(e) >= 0.f)
        kept[i * ld + id] = T(at_target(rs, 1.f, rt.put(e), caught[tg.one ? i : (int64_t)i * sp.k + tg.rank[(int64_t)i * sp.k + e]]));
    }
  }
}

// Gradients of losses per row, normaliser and targets' logits kept: what the
// logits' epilogue (S/alpha) or the passes over them (planes) need of each
// row; pad rows 0. One wave per row.
template <class O>
__global__ void __launch_bounds__(256) row_slopes_kernel(Chunk ch, LossSpec sp, Targets tg, const float* __restrict__ z,
                                                         const float2* __restrict__ norms,
                                                         const float* __restrict__ grad_rows, float scale,
                                                         const float* __restrict__ alpha, RowsOut out) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= ch.padded()) return;
  if (i >= ch.live()) {
    if (lane == 0) out.slope[i] = RowSlope{0.f, 0.f, 0.f};
    return;
  }
  const int64_t at = ch.base + i, row = ch.list[at];
  const RowTargets rt{tg, at, row, sp.k};
  const float* zr = z + at * sp.k;
  const float2 norm = norms[at];
  float qz = 0.f;
  for (int e = lane; e < sp.k; e += 64)
    if (rt.id(e) != -1) qz += rt.q(e) * (zr[e] - norm.x);
  qz = wave_sum(qz);
  const float a = grad_rows[row] * scale;
  if constexpr (kPlanes<O>) {
    out.put(i, sp, norm, qz, a, rt, zr, lane, 64);
  } else if (lane == 0) {
    out.slope[i] = row_slope(sp, norm, qz, a / alpha[0]);
    out.a[i] = a / alpha[0];
  }
}
template <typename T>
__global__ void __launch_bounds__(64) put_targets_kernel(Chunk ch, int k, Targets tg, const float* __restrict__ z,
                                                         RowsOut rows, T* __restrict__ s, int64_t ld) {
  const int i = blockIdx.x;
  if (i >= ch.live()) return;
  const int64_t at = ch.base + i;
  const RowTargets t{tg, at, ch.list[at], k};
  for (int e = threadIdx.x; e < k; e += 64)
    if (t.id(e) >= 0 && t.put(e) >= 0.f) s[i * ld + t.id(e)] = T(at_target(rows.slope[i], rows.a[i], t.put(e), z[at * k + e]));
}

// The loss of the call: a sum in a fixed order, over the count for the mean
// (no row counts: 0). A launch of its own (4 us): a counter that lets the last
// finish workgroup do it costs every one a release, which writes an XCD's L2
// back (8192 rows of 32000: +450 us).
__global__ void __launch_bounds__(1024) reduce_loss_kernel(const float* __restrict__ losses, int64_t rows,
                                                           const int* __restrict__ count, int mean,
                                                           float* __restrict__ out) {
  __shared__ double red[1024];
  double s = 0;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < rows; r += 1024) s += losses[r];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 512; w > 0; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[0] = (float)(red[0] / (mean ? max(1, count[0]) : 1));
}

// S/a and a·H as split planes for the gradients' products. dW sums over
// the rows, so a column of each has an exponent of its own, from its largest
// value: tokens that are unlikely in every row keep their bits. dH sums over
// the vocabulary, with the columns' exponents taken out of W's rows (undo); a,
// which may differ by rows, multiplies its result.

// Largest values of columns over parts of the rows, parts[part][cols]: of S/a
// (EXP, x = the logits) or of a·x. `across` threads (a power of two) take four
// columns each, and the 256/across groups of them kPartRows rows each. Bound by
// reading x (2048 x 32001: 70 us, 3.8 TB/s); the maxima cannot come with the
// logits, since a token's largest p is known only after the rows' normalisers.
constexpr int kPartRows = 64;
template <bool EXP>
__global__ void __launch_bounds__(256) column_max_kernel(Chunk ch, const float* __restrict__ x, int64_t ld, int rows,
                                                         int cols, int across, const RowSlope* __restrict__ slope,
                                                         const float* __restrict__ a, float* __restrict__ parts) {
  __shared__ float part[256][4];
  const int tid = threadIdx.x, groups = 256 / across, group = tid / across;
  const int c = (blockIdx.y * across + tid % across) * 4;
  const int r0 = (blockIdx.x * groups + group) * kPartRows, r1 = min(r0 + kPartRows, min(rows, ch.live()));
  float m[4] = {0.f, 0.f, 0.f, 0.f};
  auto take = [&](int i, const float (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = fabsf(EXP ? fmaf(slope[i].pa, pow2(v[k] - slope[i].m), slope[i].pu) : a[i] * v[k]);
      m[k] = w < INFINITY ? fmaxf(m[k], w) : m[k];
    }
  };
  // eight rows' loads in flight
  int i = c < cols ? r0 : r1;
  if (cols - c >= 4)
    for (; i + 8 <= r1; i += 8) {
      uint4 u[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) u[q] = ld16(x + (i + q) * ld + c);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        take(i + q, {__uint_as_float(u[q].x), __uint_as_float(u[q].y), __uint_as_float(u[q].z), __uint_as_float(u[q].w)});
    }
  for (; i < r1; ++i) {
    float v[4];
    load_columns(x + i * ld + c, cols - c, v);
    take(i, v);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) part[tid][k] = m[k];
  __syncthreads();
  if (group != 0 || c >= cols) return;
  for (int g = 1; g < groups; ++g)
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = fmaxf(m[k], part[g * across + tid][k]);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (c + k < cols) parts[(int64_t)blockIdx.x * cols + c + k] = m[k];
}
// Exponents of n columns (pads to np: none) from the parts' maxima and, not
// null, more of them; undo: 2^-e. 32 columns a workgroup.
__global__ void __launch_bounds__(256) exponents_kernel(const float* __restrict__ parts, int count,
                                                        const unsigned* __restrict__ more, int n, int np,
                                                        int* __restrict__ e, float* __restrict__ undo) {
  __shared__ float red[8][32];
  const int g = threadIdx.x >> 5, c = blockIdx.x * 32 + (threadIdx.x & 31);
  float m = 0.f;
  if (c < n) {
    if (more && g == 0) m = __uint_as_float(more[c]);
#pragma unroll 8
    for (int p = g; p < count; p += 8) m = fmaxf(m, parts[(int64_t)p * n + c]);
  }
  red[g][threadIdx.x & 31] = m;
  __syncthreads();
  if (g != 0 || c >= np) return;
  for (int o = 1; o < 8; ++o) m = fmaxf(m, red[o][threadIdx.x]);
  e[c] = split_exp(m);
  if (undo) undo[c] = ldexpf(1.f, -e[c]);
}
// The planes, pad rows and columns 0: S/a by workgroups (y) with runs of a
// row's columns, a·x by a wave per row. Bound by memory (S/a of 2048 x 32001:
// 122 us for 524 MB).
template <bool EXP>
__global__ void __launch_bounds__(256) column_planes_kernel(Chunk ch, const float* __restrict__ x, int64_t ld, int rows,
                                                            int cols, const RowSlope* __restrict__ slope,
                                                            const float* __restrict__ a, const int* __restrict__ ec,
                                                            sp16* __restrict__ out, int64_t ldo, int64_t pl, int k,
                                                            Targets tg, const float* __restrict__ z) {
  const int tid = threadIdx.x, i = EXP ? blockIdx.x : blockIdx.x * 4 + (tid >> 6);
  if (i >= min(rows, ch.padded())) return;
  const int64_t units = ldo / 8;
  const int64_t c0 = EXP ? units * blockIdx.y / gridDim.y * 8 : 0, c1 = EXP ? units * (blockIdx.y + 1) / gridDim.y * 8 : ldo;
  const bool live = i < ch.live();
  sp16* o = out + i * ldo;
  const RowSlope rs = EXP && live ? slope[i] : RowSlope{0.f, 0.f, 0.f};
  const float ai = !EXP && live ? a[i] : 0.f;
  constexpr int STEP = EXP ? 2048 : 512;
  auto put = [&](int64_t c, const uint4& lo, const uint4& hi, const int4& e0, const int4& e1) {
    const unsigned u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const int e[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float y = __uint_as_float(u[k]), w = EXP ? fmaf(rs.pa, pow2(y - rs.m), rs.pu) : ai * y;
      v[k] = c + k < cols ? ldexpf(w, e[k]) : 0.f;
    }
    const Split8 s = split8(v);
    *reinterpret_cast<uint4*>(o + c) = s.h;
    *reinterpret_cast<uint4*>(o + pl + c) = s.l;
  };
  int64_t c = c0 + (EXP ? tid : tid & 63) * 8;
  if (live) {
    const float* xr = x + i * ld;
    // two runs' loads in flight
    for (; c + STEP + 8 <= min(c1, (int64_t)cols); c += 2 * STEP) {
      uint4 u[4];
      int4 e[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t at = c + (q >> 1) * STEP + (q & 1) * 4;
        u[q] = ld16(xr + at);
        e[q] = *reinterpret_cast<const int4*>(ec + at);
      }
      put(c, u[0], u[1], e[0], e[1]);
      put(c + STEP, u[2], u[3], e[2], e[3]);
    }
    for (; c < min(c1, (int64_t)cols); c += STEP) {
      float lo[4], hi[4];
      load_columns(xr + c, cols - (int)c, lo);
      load_columns(xr + c + 4, cols - (int)c - 4, hi);
      uint4 u[2];
      __builtin_memcpy(&u[0], lo, 16);
      __builtin_memcpy(&u[1], hi, 16);
      put(c, u[0], u[1], *reinterpret_cast<const int4*>(ec + c), *reinterpret_cast<const int4*>(ec + c + 4));
    }
  }
  for (; c < c1; c += STEP) {
    *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(o + pl + c) = make_uint4(0, 0, 0, 0);
  }
  if constexpr (EXP) {
    if (!live) return;
    __syncthreads();  // the dense part is written before the targets' entries replace theirs
    const int64_t at = ch.base + i;
    const RowTargets rt{tg, at, ch.list[at], k};
    for (int e = tid; e < k; e += 256) {
      const int id = rt.id(e);
      if (id < c0 || id >= c1 || !(rt.put(e) >= 0.f)) continue;
      const float w = ldexpf(at_target(rs, 1.f, rt.put(e), z[at * k + e]), ec[id]);
      const _Float16 h = static_cast<_Float16>(w);
      o[id].v = h;
      o[pl + id].v = static_cast<_Float16>(w - static_cast<float>(h));
    }
  }
}

// ------------------------------------------------------------ gradients

// What a tile's values become (EpiSplit drives them): adjust as in gemm_nt.h,
// load what an output run needs, put it.
struct EpiPlain {
  typedef float S;
  typedef NoPre Pre;
  __device__ __forceinline__ void load(int, int, int, int, int, Pre&) const {}
};

// dH: rows of the chunk to their places, times what S is without: alpha, or
// each row's a (planes).
template <class O>
struct EpiRows : EpiPlain {
  typedef Elem<O> T;
  Chunk ch;
  T* dst;
  int64_t ld;
  const float* a;
  __device__ __forceinline__ bool adjust(GemmArgs& g, int, int row0, int) const {
    g.M = ch.live();
    return row0 < g.M;
  }
  __device__ __forceinline__ void put(int, int i, int j0, const S* v, int kbeg, int n, const Pre&, S*) const {
    const float f = a[kPlanes<O> ? i : 0];
    S w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = v[k] * f;
    st8<T, S>(dst + ch.list[ch.base + i] * ld + j0, w, kbeg, n);
  }
};

// dW over the chunks of rows: acc = v (first), acc + v, and out = acc + v,
// times alpha (S of planes is without each row's a, which H has) and rounded
// (last); acc is out where the chunk is the only one or out is fp32.
template <class O>
struct EpiWeight : EpiPlain {
  typedef Elem<O> T;
  Chunk ch;
  float* acc;
  T* out;
  int64_t ld;
  int first, last;
  const float* alpha;
  typedef Raw8<float> Pre;
  __device__ __forceinline__ bool adjust(GemmArgs& g, int, int, int) const {
    // fp32: rows as far as its rings of K tiles (64)
    g.K = std::is_same<O, float>::value ? (ch.live() + 63) / 64 * 64 : ch.padded();
    return g.K > 0 || first || last;
  }
  __device__ __forceinline__ void load(int, int i, int j0, int kbeg, int n, Pre& p) const {
    if (!first) ld8_pre<float>(acc + i * ld + j0, p, kbeg, n);
  }
  __device__ __forceinline__ void put(int, int i, int j0, const S* v, int kbeg, int n, const Pre& p, S*) const {
    float r[8];
    if (first) {
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = v[k];
    } else {
      ld8_use<float, float>(acc + i * ld + j0, p, r, kbeg, n);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] += v[k];
    }
    if (last && !kPlanes<O>) {
      const float f = alpha[0];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] *= f;
    }
    if (last)
      st8<T, float>(out + i * ld + j0, r, kbeg, n);
    else
      st8<float, float>(acc + i * ld + j0, r, kbeg, n);
  }
};

// One of them over split operands: the powers of two of the rows (er, or none)
// and columns taken out first.
template <class In>
struct EpiPowers : EpiPlain {
  typedef typename In::Pre Pre;
  In in;
  const int *er, *ec;
  int off;
  __device__ __forceinline__ bool adjust(GemmArgs& g, int b, int row0, int col0) const {
    return in.adjust(g, b, row0, col0);
  }
  __device__ __forceinline__ void load(int b, int i, int j0, int kbeg, int n, Pre& p) const {
    in.load(b, i, j0, kbeg, n, p);
  }
  __device__ __forceinline__ void put(int b, int i, int j0, const S* v, int kbeg, int n, const Pre& p, S*) const {
    S w[8], drop[8];
    const int e = off - (er ? er[i] : 0);
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = k < n ? ldexpf(v[k], e - ec[j0 + k]) : 0.f;
    in.put(b, i, j0, w, kbeg, n, p, drop);
  }
};

// Parts of K for the tiles that whole rounds of the CUs leave over: as many as
// end soonest, with `unit` us for kPadK of K of a tile on one CU and the
// partial tiles' way to memory and back (`area` elements) against it. How many
// tiles there are only the device knows (rows left out), so the choice is made
// there, by every workgroup alike.
struct Parts {
  int full, rest, parts;  // tiles in whole rounds, tiles left over, parts of each of those
  float time;
};
constexpr int kMostParts = 128;
struct TileTime {
  float unit, fixed;
};
__host__ __device__ inline Parts split_parts(int tiles, int units, int cus, TileTime tt, int area, int most) {
  Parts s;
  s.full = tiles / cus * cus;
  s.rest = tiles - s.full;
  s.parts = 1;
  s.time = s.rest > 0 ? units * tt.unit + tt.fixed : 0.f;
  // 2, 3, 4, 6, 8, 12, ...
  for (int p = 2; p <= most && p <= units && s.rest > 0 && s.rest * p <= 2 * cus; p += (p & (p - 1)) ? p / 3 : p / 2) {
    const float t = (float)((s.rest * p + cus - 1) / cus) * ((units + p - 1) / p * tt.unit + tt.fixed) + 7.f +
                    (float)s.rest * p * area * (8.f / 4.5e6f);
    if (t < s.time) {
      s.time = t;
      s.parts = p;
    }
  }
  return s;
}

// Any of them, with the tiles of the last round in parts: partial tiles to the
// workspace, joined by join_parts_kernel. 8192 x 2048 x 32000: dH 857 us, dW
// 856, 1.25 PFLOP/s, at the board's power limit.
template <class In, class Cfg, bool QN, bool PT, typename T, bool TAIL>
struct EpiSplit {
  typedef float S;
  typedef typename In::Pre Pre;
  typedef NoPre PreT;
  static constexpr bool kVoIsV = true;
  static constexpr int BM = Cfg::BM, BN = Cfg::BN;
  In in;
  float* part;
  TileTime tt;
  int most, cus;
  static constexpr bool kTail = TAIL;
  int tail_k = 0;           // K from which Q's rows lie in a padded copy
  int64_t tail_bytes_ = 0;  // and how far from their place
  int slot = -1, row0 = 0, col0 = 0;
  __device__ __forceinline__ int tail_tile() const { return tail_k / Cfg::BK; }
  __device__ __forceinline__ int64_t tail_bytes() const { return tail_bytes_; }
  struct Plan {
    Parts s;
    int tm, tn, units;
  };
  __device__ __forceinline__ bool plan(GemmArgs& g, Plan& p) const {
    if (!in.adjust(g, 0, 0, 0)) return false;
    p.tm = (g.M + BM - 1) / BM;
    p.tn = (g.N + BN - 1) / BN;
    p.units = g.K / kPadK;
    p.s = split_parts(p.tm * p.tn, p.units, cus, tt, BM * BN, most);
    return true;
  }
  __device__ __forceinline__ int work(const GemmArgs& g0) const {
    GemmArgs g = g0;
    Plan p;
    return plan(g, p) ? p.s.full + p.s.rest * p.s.parts : 0;
  }
  __device__ __forceinline__ bool take(GemmArgs& g, int logical, int& ti, int& tj) {
    Plan p;
    plan(g, p);
    int tile = logical;
    if (logical >= p.s.full && p.s.parts > 1) {
      slot = logical - p.s.full;
      tile = p.s.full + slot / p.s.parts;
      const int of = slot % p.s.parts, k0 = p.units * of / p.s.parts * kPadK;
      g.K = p.units * (of + 1) / p.s.parts * kPadK - k0;
      g.P = static_cast<const T*>(g.P) + (PT ? k0 * g.ldp : k0);
      g.Q = static_cast<const T*>(g.Q) + (QN ? k0 * g.ldq : k0);
      tail_k -= k0;
    }
    decode_tile<false>(tile, p.tm, p.tn, ti, tj);
    row0 = ti * BM;
    col0 = tj * BN;
    return true;
  }
  __device__ __forceinline__ bool has_t() const { return false; }
  __device__ __forceinline__ void load(int b, int i, int j0, int kbeg, int n, Pre& p, bool = false) const {
    if (slot < 0) in.load(b, i, j0, kbeg, n, p);
  }
  __device__ __forceinline__ void load_t(int, int, int, int, PreT&, bool = false) const {}
  __device__ __forceinline__ void put_t(int, int, int, const S*, int, const PreT&, bool = false) const {}
  __device__ __forceinline__ void finish(int) const {}
  __device__ __forceinline__ void put(int b, int i, int j0, const S* v, int kbeg, int n, const Pre& p, S* vo,
                                      bool = false) const {
    if (slot < 0)
      in.put(b, i, j0, v, kbeg, n, p, vo);
    else
      st8<float, S>(part + ((int64_t)slot * BM + (i - row0)) * BN + (j0 - col0), v, kbeg, n);
  }
};

// 16 rows of a tile in parts a workgroup.
template <class Epi>
__global__ void __launch_bounds__(256) join_parts_kernel(GemmArgs g, Epi epi) {
  constexpr int BM = Epi::BM, BN = Epi::BN, RUNS = BN / 8;
  typename Epi::Plan p;
  if (!epi.plan(g, p) || p.s.parts == 1 || (int)blockIdx.x >= p.s.rest) return;
  int ti, tj;
  decode_tile<false>(p.s.full + blockIdx.x, p.tm, p.tn, ti, tj);
  const float* part = epi.part + (int64_t)blockIdx.x * p.s.parts * BM * BN;
#pragma unroll
  for (int q = threadIdx.x; q < 16 * RUNS; q += 256) {
    const int r = blockIdx.y * 16 + q / RUNS, c = q % RUNS * 8, i = ti * BM + r, j0 = tj * BN + c;
    const int n = min(8, g.N - j0);
    if (i >= g.M || n <= 0) continue;
    typename Epi::Pre pre;
    epi.in.load(0, i, j0, 0, n, pre);
    float v[8] = {}, drop[8];
#pragma unroll 4
    for (int k = 0; k < p.s.parts; ++k) {
      const float4* x = reinterpret_cast<const float4*>(part + ((int64_t)k * BM + r) * BN + c);
      const float4 lo = x[0], hi = x[1];
      v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
      v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
    }
    epi.in.put(0, i, j0, v, 0, n, pre, drop);
  }
}

// x and y *= s[0] in place, nothing read where s[0] is 1 (the gradients of a
// loss that is itself differentiated).
template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(T* __restrict__ x, int64_t n, T* __restrict__ y, int64_t m,
                                                    const float* __restrict__ s) {
  const float f = s[0];
  if (f == 1.f) return;
  constexpr int E = 16 / (int)sizeof(T);
  const int64_t step = (int64_t)gridDim.x * 256 * E, first = ((int64_t)blockIdx.x * 256 + threadIdx.x) * E;
  auto run = [&](T* p, int64_t len) {
    for (int64_t c = first; c < len; c += step) {
      if (c + E <= len) {
        uint4 u = ld16(p + c);
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int k = 0; k < E; ++k) e[k] = convert<T>(to_f(e[k]) * f);
        st16(p + c, u);
      } else {
        for (int64_t k = c; k < len; ++k) p[k] = convert<T>(to_f(p[k]) * f);
      }
    }
  };
  run(x, n);
  run(y, m);
}

// ------------------------------------------------------------ host

struct Call {
  const void* h;
  int64_t ldh;
  const void* w;
  int64_t ldw;
  bool kd;
  const int64_t* y;       // cross entropy
  int64_t ignore;
  const float* teacher;   // distillation
  const int64_t* index;
  int64_t rows, d, vocab, k;
  double temp, smooth, zeta;
  int reduction;
  const float* grad_rows;
  float *loss, *norm, *z;
  void *dh, *dw;
  int64_t chunk_bytes;
  const char* name;
};

// Microseconds of a tile on one CU (the smaller run in twos), measured.
template <class O, class Cfg>
constexpr TileTime tile_time() {
  constexpr bool big = Cfg::BM == TileSet<O>::big::BM;
  constexpr float rate = std::is_same<O, float>::value ? 30.f : kPlanes<O> ? 8.25f : 3.6f;
  return {rate / 65536 * Cfg::BM * Cfg::BN * (big ? 1.f : (float)TileSet<O>::kBigRate),
          std::is_same<O, float>::value ? 4.f : kPlanes<O> ? (big ? 20.f : 5.f) : (big ? 11.5f : 3.5f)};
}
// From this many rounds of tiles on, the last one is not worth parts.
constexpr int kWholeRounds = 12;
constexpr int64_t kPartFloats = 2 * 65536;  // per CU: two rounds of partial 256² tiles

template <class O, class Cfg, class In, bool QN, bool PT, bool TAIL>
int launch_gradient_cfg(const ArgsOf<O>& args, const In& in, float* part, hipStream_t s, const char* name,
                    int tail_k, const void* tail) {
  typedef EpiSplit<In, Cfg, QN, PT, O, TAIL> Epi;
  ArgsOf<O> g = args;
  PTO_REQUIRE(g.K % ring_k<O>() == 0 && g.ldq < (int64_t(1) << 26) && g.ldp < (int64_t(1) << 26) && g.ldp * sizeof(O) % 16 == 0 &&
                  g.ldq * sizeof(O) % 16 == 0 && (!QN || g.ldq >= g.N) && (!PT || g.ldp >= g.M) &&
                  ((reinterpret_cast<uintptr_t>(g.P) | reinterpret_cast<uintptr_t>(g.Q)) & 15) == 0,
              std::string(name) + ": operands not padded or not 16-byte aligned");
  g.tiles_m = (g.M + Cfg::BM - 1) / Cfg::BM;
  g.tiles_n = (g.N + Cfg::BN - 1) / Cfg::BN;
  g.cus = device_cus();
  const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n;
  if (tiles == 0) return 0;
  // dW's tiles are known here, and fewer rows make parts pay less
  const bool whole = tiles >= kWholeRounds * g.cus ||
                     (PT && split_parts((int)tiles, g.K / kPadK, g.cus, tile_time<O, Cfg>(), Cfg::BM * Cfg::BN,
                                        kMostParts).parts == 1);
  Epi e{in, part, tile_time<O, Cfg>(), whole ? 1 : kMostParts, g.cus};
  if (TAIL) {
    e.tail_k = tail_k;
    e.tail_bytes_ = static_cast<const char*>(tail) - static_cast<const char*>(g.Q) - (int64_t)tail_k * g.ldq * (int64_t)sizeof(O);
  }
  const int64_t grid = tiles + (e.most > 1 ? 2 * g.cus : 0);
  PTO_REQUIRE(grid < (1ll << 31), std::string(name) + ": grid too large");
  ProfScope ps(name, s);
  hipLaunchKernelGGL((gemm_nt_kernel<O, Cfg, false, Epi, QN, PT, false, ArgsOf<O>>), dim3((unsigned)grid), dim3(Cfg::NT),
                     0, s, g, e);
  PTO_LAUNCHED(name);
  if (e.most > 1) {
    hipLaunchKernelGGL(join_parts_kernel<Epi>, dim3((unsigned)std::min<int64_t>(tiles, g.cus), Cfg::BM / 16), dim3(256),
                       0, s, static_cast<const GemmArgs&>(g), e);
    PTO_LAUNCHED("join_parts");
  }
  return 0;
}
// With the tile that ends sooner if every row counts.
template <class O, bool QN, bool PT, class In>
int launch_gradient(const ArgsOf<O>& g, const In& in, float* part, hipStream_t s, const char* name,
                    int tail_k = 0, const void* tail = nullptr) {
  // dW of few fp32 rows is mostly written, and five workgroups a CU write it 3%
  // (3584 x 21675) to 5% (1024 x 32000) sooner than two of 128² tiles
  if constexpr (std::is_same<O, float>::value && PT)
    return launch_gradient_cfg<O, Tile<64, 64, 16, 2, 2>, In, QN, PT, false>(g, in, part, s, name, 0, nullptr);
  typedef typename TileSet<O>::big Big;
  typedef typename TileSet<O>::small Small;
  const int cus = device_cus(), units = g.K / kPadK;
  auto time = [&](int bm, int bn, TileTime tt) {
    const int tiles = ((g.M + bm - 1) / bm) * ((g.N + bn - 1) / bn);
    const Parts p = split_parts(tiles, units, cus, tt, bm * bn, kMostParts);
    return p.time + (float)(p.full / cus) * (units * tt.unit + tt.fixed);
  };
  const bool big = time(Big::BM, Big::BN, tile_time<O, Big>()) <= time(Small::BM, Small::BN, tile_time<O, Small>());
  if constexpr (QN && !PT && !kPlanes<O>) {
    if (tail)
      return big ? launch_gradient_cfg<O, Big, In, QN, PT, true>(g, in, part, s, name, tail_k, tail)
                 : launch_gradient_cfg<O, Small, In, QN, PT, true>(g, in, part, s, name, tail_k, tail);
  }
  return big ? launch_gradient_cfg<O, Big, In, QN, PT, false>(g, in, part, s, name, 0, nullptr)
             : launch_gradient_cfg<O, Small, In, QN, PT, false>(g, in, part, s, name, 0, nullptr);
}

// Whether the products (not of planes) read W where it lies, else from a padded copy. They can
// where its rows are 16-byte aligned and what follows a row's end up to a
// multiple of kPadK is nothing but the next row (an infinity there times H's
// zero makes a NaN of a row that it would have made infinite itself), and do
// where nothing needs padding or the rows of H are few. Copying costs a read and
// a write of W, 5001 x 1000 x 50001 (2000 rows count) 32 us; reading in place
// rows that are no whole 128-byte lines 50, a tail of the vocabulary 5% of dH
// (8192 x 2048 x 32000: 15 against 53 for the copy, 64 x 2240 x 35072: 2
// against 52).
inline bool reads_in_place(const Call& c, int64_t dp, int64_t element) {
  if (c.ldw * element % 16 || (c.d % kPadK && (c.ldw != c.d || dp - c.d > c.d))) return false;
  return (c.d % kPadK == 0 && (!c.dh || c.vocab % kPadK == 0)) || c.rows <= (c.ldw * element % 128 ? 1024 : 8192);
}

template <class O>
struct Ws {
  typedef Elem<O> T;
  static constexpr bool planes = kPlanes<O>;
  int64_t dp, vp, blocks, cap, capp;
  bool pad_w, in_place;
  Targets t{};
  int *list, *count;
  T* hc;
  // W padded; or its last rows up to a multiple of kPadK and, by itself,
  // its last one
  T *wp, *tail, *last;
  float2 *stats, *norm;
  float *sums, *losses, *z, *caught, *alpha;
  RowsOut rows;
  T* kept;  // the kept logits; not of planes: then S
  // Planes of H and W (by rows) for the logits, of S/a, W (S's exponents
  // taken out) and a·H (by columns) for the gradients
  sp16 *hp, *wpl, *sp, *ws, *ah;
  int *eh, *ew, *es, *ews, *eah;  // es, ews and eah: exponents of the columns' maxima
  float *undo, *parts;  // 2^-es; maxima of parts of the rows
  float *part, *acc;
  int64_t chunks(const Call& c) const { return c.rows ? (c.rows + cap - 1) / cap : 0; }
  Ws(Carver& cv, const Call& c) {
    const bool grads = c.dh || c.dw;
    dp = round_up(c.d, kPadK);
    vp = round_up(c.vocab, kPadK);
    blocks = vp / kCols;
    const int64_t per = grads ? vp * (planes ? 8 : (int64_t)sizeof(T)) : blocks * 8;
    cap = (c.chunk_bytes > 0 ? c.chunk_bytes : kChunkBytes) / per;
    cap = std::min(std::max<int64_t>(cap / 256 * 256, 256), std::max<int64_t>(c.rows, 1));
    capp = round_up(cap, kPadK);
    pad_w = !planes && !reads_in_place(c, dp, sizeof(T));
    const bool join = !c.grad_rows;
    if (c.kd) {
      t.id = cv.take<int>(c.rows * c.k);
      t.q = cv.take<float>(c.rows * c.k);
      t.put = cv.take<float>(c.rows * c.k);
      t.entropy = cv.take<float>(c.rows);
      t.kept = cv.take<int>(c.rows);
      t.rank = cv.take<uint16_t>(cap * c.k);
    } else {
      t.one = cv.take<int>(c.rows);
      t.share = (float)(1.0 - c.smooth);
    }
    if (c.kd && join) {
      t.bits = cv.take<unsigned long long>(blocks * cap);
      t.before = cv.take<uint16_t>(blocks * cap);
    }
    list = cv.take<int>(c.rows);
    count = cv.take<int>(4);
    alpha = cv.take<float>(4);
    // scoring reads aligned rows of H where they lie
    in_place = !planes && !grads && c.h && c.d % kPadK == 0 && c.ldh * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(c.h) & 15) == 0;
    hc = in_place ? nullptr : cv.take<T>(capp * dp);
    wp = pad_w ? cv.take<T>(vp * dp) : nullptr;
    tail = !planes && !pad_w && c.dh && c.vocab % kPadK ? cv.take<T>(kPadK * c.ldw) : nullptr;
    last = !planes && !pad_w && c.d % kPadK ? cv.take<T>(dp) : nullptr;
    losses = cv.take<float>(c.rows);
    norm = cv.take<float2>(c.rows);
    z = cv.take<float>(c.rows * c.k);
    caught = join ? cv.take<float>(cap * c.k) : nullptr;
    stats = join || planes ? cv.take<float2>(cap * blocks) : nullptr;
    sums = c.smooth != 0 && join ? cv.take<float>(cap * blocks) : nullptr;
    rows = RowsOut{grads && (planes || c.grad_rows) ? cv.take<RowSlope>(capp) : nullptr,
                   grads && (planes || c.grad_rows) ? cv.take<float>(capp) : nullptr, nullptr};
    kept = grads ? cv.take<T>(capp * vp) : nullptr;
    hp = wpl = sp = ws = ah = nullptr;
    eh = ew = es = ews = eah = nullptr;
    undo = parts = nullptr;
    if (planes) {
      hp = cv.take<sp16>(2 * capp * dp);
      wpl = cv.take<sp16>(2 * c.vocab * dp);
      eh = cv.take<int>(capp);
      ew = cv.take<int>(c.vocab);
    }
    if (planes && grads) {
      rows.maxima = cv.take<unsigned>(vp);
      es = cv.take<int>(vp + 2 * dp);
      eah = es + vp;
      ews = eah + dp;
      parts = cv.take<float>(std::max((cap + kPartRows - 1) / kPartRows * vp, (c.vocab + kPartRows - 1) / kPartRows * dp));
      sp = cv.take<sp16>(2 * capp * vp);
      if (c.dw) ah = cv.take<sp16>(2 * capp * dp);
      if (c.dh) {
        ws = cv.take<sp16>(2 * vp * dp);
        undo = cv.take<float>(vp);
      }
    }
    part = grads ? cv.take<float>(kPartFloats * device_cus()) : nullptr;
    acc = sizeof(T) == 2 && c.dw && chunks(c) > 1 ? cv.take<float>(c.vocab * c.d) : nullptr;
  }
};

template <class O>
size_t loss_ws_bytes(const Call& c) {
  Carver cv(nullptr, 0);
  Ws<O> w(cv, c);
  return cv.used + 512;
}

// Whether fp32 products run on fp32's own matrix instructions, a third of the
// planes' rate, but W's bytes are read twice, where the planes read or write
// them seven times. Losses and gradients of 64 x 3584 x 21675 take 415 us
// (planes: 838), 128 x 1024 x 32000 283 (412); at 192 rows one or the other is
// 13% faster by shape, at 256 the planes by up to 20%. A padded copy of W costs
// scores as much as their planes.
inline bool few_rows(const Call& c) {
  return c.rows <= kPadK && (c.dh || c.dw || reads_in_place(c, round_up(c.d, kPadK), 4));
}

// Workgroups per row of `cols`: two per CU in all, 2048 columns each at least.
inline unsigned segments(int64_t rows, int64_t cols) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(2 * device_cus() / rows, cols / 2048));
}

// The logits' product: two sizes of tile, both of 64-column wave tiles.
template <class O, class Epi>
int launch_logits(const ArgsOf<O>& g, const Epi& e, hipStream_t s) {
  typedef typename TileSet<O>::big Big;
  typedef std::conditional_t<std::is_same<O, float>::value, Tile<64, 64, 16, 4, 1, 8>, Tile<128, 128, 32, 2, 2>> Small;
  const int64_t cus = device_cus();
  auto time = [&](int64_t b, TileTime tt) {
    return double(((g.M + b - 1) / b * ((g.N + b - 1) / b) + cus - 1) / cus) * (g.K / kPadK * tt.unit + tt.fixed);
  };
  if (time(Big::BM, tile_time<O, Big>()) <= time(Small::BM, tile_time<O, Small>()))
    return launch_gemm_cfg<O, Big, false>(g, e, 1, s, "loss_logits");
  return launch_gemm_cfg<O, Small, false>(g, e, 1, s, "loss_logits");
}

// dH and dW of a chunk from its S.
template <class O>
int chunk_gradients(const Call& c, const Ws<O>& w, const Chunk& ch, const O* W, int64_t ldw, bool first, bool last,
                    hipStream_t s) {
  if (c.dh && ch.cap > 0) {
    const GemmArgs g{w.kept, w.vp, 0, W, ldw, 0, ch.cap, (int)c.d, (int)w.vp, 0, 0, nullptr};
    const EpiRows<O> e{{}, ch, static_cast<O*>(c.dh), c.d, w.alpha};
    if (launch_gradient<O, true, false>(g, e, w.part, s, "loss_dhidden", (int)(c.vocab / kPadK * kPadK), w.tail))
      return -1;
  }
  if (c.dw) {
    const int k = (int)round_up(ch.cap, kPadK);
    const GemmArgs g{w.kept, w.vp, 0, w.hc, w.dp, 0, (int)c.vocab, (int)c.d, k, 0, 0, nullptr};
    float* acc = w.acc;
    if constexpr (sizeof(O) == 4) acc = static_cast<float*>(c.dw);
    const EpiWeight<O> e{{}, ch, acc, static_cast<O*>(c.dw), c.d, first, last, w.alpha};
    if (launch_gradient<O, true, true>(g, e, w.part, s, "loss_dweight")) return -1;
  }
  return 0;
}

int chunk_gradients(const Call& c, const Ws<sp16>& w, const Chunk& ch, const LossSpec& sp, const float* z, bool first,
                    bool last, hipStream_t s) {
  float *dh = static_cast<float*>(c.dh), *dw = static_cast<float*>(c.dw);
  const int k = (int)round_up(ch.cap, kPadK), cap = ch.cap, vocab = (int)c.vocab, d = (int)c.d;
  // the exponents of the columns (np with pads) of S/a or a·x
  auto exponents = [&](auto exp, const Chunk& of, const float* x, int64_t ld, int rows, int cols, int64_t np,
                       const float* a, int* e, float* undo) {
    int across = 256;
    while (across > 16 && across * 2 >= cols) across /= 2;
    const int each = 256 / across * kPartRows, count = (rows + each - 1) / each;
    hipLaunchKernelGGL((column_max_kernel<decltype(exp)::value>),
                       dim3((unsigned)count, (unsigned)((cols + across * 4 - 1) / (across * 4))), dim3(256), 0, s, of, x,
                       ld, rows, cols, across, w.rows.slope, a, w.parts);
    PTO_LAUNCHED("column_max");
    hipLaunchKernelGGL(exponents_kernel, dim3((unsigned)((np + 31) / 32)), dim3(256), 0, s, w.parts, count,
                       decltype(exp)::value ? w.rows.maxima : nullptr, cols, (int)np, e, undo);
    PTO_LAUNCHED("exponents");
    return 0;
  };
  if (cap > 0) {
    if (exponents(std::true_type{}, ch, w.kept, w.vp, cap, vocab, w.vp, w.rows.a, w.es, w.undo)) return -1;
    if (dw && exponents(std::false_type{}, ch, w.hc, w.dp, cap, d, w.dp, w.rows.a, w.eah, nullptr)) return -1;
    hipLaunchKernelGGL(column_planes_kernel<true>, dim3((unsigned)k, segments(k, w.vp)), dim3(256), 0, s, ch, w.kept, w.vp, k, vocab,
                       w.rows.slope, w.rows.a, w.es, w.sp, w.vp, w.capp * w.vp, sp.k, w.t, z);
    PTO_LAUNCHED("column_planes");
  }
  if (dh && cap > 0) {
    const Chunk all{nullptr, nullptr, 0, 0, vocab};
    const float* W = static_cast<const float*>(c.w);
    if (exponents(std::false_type{}, all, W, c.ldw, vocab, d, w.dp, w.undo, w.ews, nullptr)) return -1;
    hipLaunchKernelGGL(column_planes_kernel<false>, dim3((unsigned)(w.vp / 4)), dim3(256), 0, s, all, W, c.ldw, (int)w.vp, d,
                       w.rows.slope, w.undo, w.ews, w.ws, w.dp, w.vp * w.dp, sp.k, w.t, z);
    PTO_LAUNCHED("column_planes");
    const SplitArgs g{{w.sp, w.vp, 0, w.ws, w.dp, 0, cap, d, (int)w.vp}, w.capp * w.vp, w.vp * w.dp};
    const EpiPowers<EpiRows<sp16>> e{{}, {{}, ch, dh, c.d, w.rows.a}, nullptr, w.ews, 0};
    if (launch_gradient<sp16, true, false>(g, e, w.part, s, "loss_dhidden")) return -1;
  }
  if (dw) {
    if (cap > 0) {
      hipLaunchKernelGGL(column_planes_kernel<false>, dim3((unsigned)(k / 4)), dim3(256), 0, s, ch, w.hc, w.dp, k, d,
                         w.rows.slope, w.rows.a, w.eah, w.ah, w.dp, w.capp * w.dp, sp.k, w.t, z);
      PTO_LAUNCHED("column_planes");
    }
    const SplitArgs g{{w.sp, w.vp, 0, w.ah, w.dp, 0, vocab, d, k}, w.capp * w.vp, w.capp * w.dp};
    const EpiPowers<EpiWeight<sp16>> e{{}, {{}, ch, dw, dw, c.d, first, last, nullptr}, w.es, w.eah, 0};
    if (launch_gradient<sp16, true, true>(g, e, w.part, s, "loss_dweight")) return -1;
  }
  return 0;
}

template <class O>
int loss_t(const Call& c, void* ws, size_t ws_bytes, hipStream_t s) {
  typedef Elem<O> T;
  constexpr bool planes = kPlanes<O>;
  Carver cv(ws, ws_bytes);
  const Ws<O> w(cv, c);
  PTO_REQUIRE(!cv.overflow, std::string(c.name) + ": workspace too small");
  const bool grads = c.dh || c.dw;
  const T* W = static_cast<const T*>(c.w);
  int64_t ldw = c.ldw;
  float2* norm = c.norm ? reinterpret_cast<float2*>(c.norm) : w.norm;
  float* z = c.z ? c.z : w.z;
  float* losses = c.reduction || !c.loss ? w.losses : c.loss;
  const float scale = (float)(1.4426950408889634 / c.temp);
  const LossSpec sp{(float)(c.temp * c.temp), (float)(c.smooth / c.vocab), (float)c.zeta, (int)c.k};
  if (c.kd && c.rows > 0) {
    hipLaunchKernelGGL(kd_targets_kernel, dim3((unsigned)((c.rows + 3) / 4)), dim3(256), 0, s, c.teacher, c.index,
                       c.rows, (int)c.k, c.vocab, (float)(1.0 / c.temp), w.t);
    PTO_LAUNCHED("kd_targets");
  }
  hipLaunchKernelGGL(list_rows_kernel, dim3(1), dim3(1024), 0, s, c.kd ? nullptr : c.y, c.ignore, c.vocab, w.t, c.rows,
                     w.list, w.count, c.grad_rows ? nullptr : losses, c.grad_rows, (float)c.temp, c.reduction == 1,
                     w.alpha);
  PTO_LAUNCHED("list_rows");
  if (c.rows > 0) {
    if constexpr (planes) {
      hipLaunchKernelGGL(weight_planes_kernel, dim3((unsigned)((c.vocab + 3) / 4)), dim3(256), 0, s, W, ldw, c.vocab,
                         c.d, w.wpl, w.dp, w.ew);
      PTO_LAUNCHED("weight_planes");
    } else if (w.pad_w) {
      hipLaunchKernelGGL(pad_weight_kernel<T>, dim3((unsigned)((w.vp + 3) / 4)), dim3(256), 0, s, W, ldw, c.vocab, c.d,
                         w.wp, w.dp, w.vp);
      PTO_LAUNCHED("pad_weight");
      W = w.wp;
      ldw = w.dp;
    } else if (w.tail || w.last) {
      hipLaunchKernelGGL(weight_tail_kernel<T>, dim3(kPadK / 4), dim3(256), 0, s, W, ldw, c.vocab, c.d, w.tail, w.last, w.dp);
      PTO_LAUNCHED("weight_tail");
    }
  }
  const int64_t chunks = std::max<int64_t>(w.chunks(c), c.dw ? 1 : 0);  // no rows: dW is still written
  for (int64_t n = 0; n < chunks; ++n) {
    const Chunk ch{w.list, w.count, c.rows, (int)(n * w.cap), (int)std::min(w.cap, c.rows - n * w.cap)};
    if (ch.cap > 0) {
      const unsigned capp = (unsigned)round_up(ch.cap, kPadK);
      GemmArgs base{w.hc, w.dp, 0, W, ldw, 0, ch.cap, (int)w.vp, (int)w.dp, 0, 0, nullptr};
      ArgsOf<O> g{base};
      if constexpr (planes) {
        hipLaunchKernelGGL(gather_planes_kernel, dim3(capp / 4), dim3(256), 0, s, ch, static_cast<const float*>(c.h),
                           c.ldh, c.d, w.hc, w.dp, w.hp, w.capp * w.dp, w.eh, static_cast<float*>(c.dh), w.rows.maxima,
                           grads ? w.vp : 0);
        g.P = w.hp;
        g.Q = w.wpl;
        g.ldq = w.dp;
        g.pP = w.capp * w.dp;
        g.pQ = c.vocab * w.dp;
      } else if (w.in_place) {
        g.P = c.h;
        g.ldp = c.ldh;
      } else {
        hipLaunchKernelGGL(gather_kernel<T>, dim3(capp / 4), dim3(256), 0, s, ch, static_cast<const T*>(c.h), c.ldh,
                           c.d, w.hc, w.dp, static_cast<T*>(c.dh));
      }
      PTO_LAUNCHED("gather");
      if (c.kd) {
        int several = 8;
        while (several > 1 && several * w.blocks * 10 > kMaxMarked / kCols * 10) several /= 2;
        hipLaunchKernelGGL(mark_targets_kernel, dim3((unsigned)((ch.cap + several - 1) / several)), dim3(256),
                           (unsigned)(several * w.blocks * 10), s, ch, (int)w.blocks, several, (int)c.k, w.t);
        PTO_LAUNCHED("mark_targets");
      }
      if (c.grad_rows) {
        hipLaunchKernelGGL(row_slopes_kernel<O>, dim3(capp / 4), dim3(256), 0, s, ch, sp, w.t, z, norm, c.grad_rows,
                           (float)c.temp, w.alpha, w.rows);
        PTO_LAUNCHED("row_slopes");
        if constexpr (planes) {
          const EpiLogits<O, true, false> e{ch,      (int)c.vocab, scale, w.stats, nullptr, w.blocks, w.kept,
                                            w.vp,    nullptr,      w.eh,  w.ew,    w.t,     sp.k,     nullptr, false,
                                            w.last};
          if (launch_logits<O>(g, e, s)) return -1;
        } else {
          g.M = (int)capp;
          const EpiLogits<O, false, true> e{ch,   (int)c.vocab, scale,   nullptr, nullptr, w.blocks, w.kept,
                                            w.vp, w.rows.slope, nullptr, nullptr, w.t,     sp.k,     nullptr, false,
                                            w.last};
          if (launch_logits<O>(g, e, s)) return -1;
          hipLaunchKernelGGL(put_targets_kernel<T>, dim3((unsigned)ch.cap), dim3(64), 0, s, ch, sp.k, w.t, z, w.rows,
                             w.kept, w.vp);
          PTO_LAUNCHED("put_targets");
        }
      } else {
        auto logits = [&](auto keep) {
          const EpiLogits<O, decltype(keep)::value, false> e{ch,     (int)c.vocab, scale, w.stats, w.sums,
                                                             w.blocks, w.kept,     w.vp,  nullptr, w.eh,
                                                             w.ew,   w.t,          sp.k,  w.caught, w.in_place,
                                                             w.last};
          return launch_logits<O>(g, e, s);
        };
        if (grads ? logits(std::true_type{}) : logits(std::false_type{})) return -1;
        hipLaunchKernelGGL((grads ? finish_kernel<O, true> : finish_kernel<O, false>),
                           dim3(capp, grads && !planes ? segments(capp, w.vp) : 1), dim3(256), 0, s, ch, w.stats, w.sums,
                           w.blocks, sp, w.t, w.caught, (int)c.vocab, w.kept, w.vp, w.rows, w.alpha, losses, norm, z);
        PTO_LAUNCHED("finish");
      }
    }
    const bool first = n == 0, last = n == chunks - 1;
    if constexpr (planes) {
      if (grads && chunk_gradients(c, w, ch, sp, z, first, last, s)) return -1;
    } else {
      if (grads && chunk_gradients(c, w, ch, W, ldw, first, last, s)) return -1;
    }
  }
  if (c.reduction && c.loss) {
    hipLaunchKernelGGL(reduce_loss_kernel, dim3(1), dim3(1024), 0, s, w.losses, c.rows, w.count, c.reduction == 1,
                       c.loss);
    PTO_LAUNCHED("reduce_loss");
  }
  return 0;
}

int check(const Call& c, int dtype, void* ws, size_t ws_bytes) {
  const std::string n(c.name);
  PTO_REQUIRE(dtype == kF32 || dtype == kBF16, n + ": unsupported dtype code (fp32 and bf16)");
  PTO_REQUIRE(c.rows >= 0 && c.d >= 1 && c.vocab >= 1, n + ": negative row count, or no features or tokens");
  PTO_REQUIRE(c.rows < (1ll << 30) && c.d < (1ll << 24) && c.vocab < (1ll << 25), n + ": shape too large");
  PTO_REQUIRE(c.k >= 1 && c.k <= kMaxTeach && c.rows * c.k < (1ll << 32), n + ": 1 to 1024 teacher entries per row");
  PTO_REQUIRE(c.ldh >= c.d && c.ldw >= c.d, n + ": row pitch below the width");
  PTO_REQUIRE(c.ldw < (int64_t(1) << 26), n + ": row pitch too large");
  PTO_REQUIRE(c.reduction >= 0 && c.reduction <= 2, n + ": reduction is 0 (none), 1 (mean) or 2 (sum)");
  PTO_REQUIRE(c.temp > 0 && std::isfinite(c.temp), n + ": temperature must be positive");
  PTO_REQUIRE(c.smooth >= 0 && c.smooth <= 1, n + ": label smoothing outside [0, 1]");
  PTO_REQUIRE(std::isfinite(c.zeta), n + ": z_loss must be finite");
  PTO_REQUIRE(c.w && (c.rows == 0 || (c.h && (c.y || (c.teacher && c.index)))), n + ": null operand");
  PTO_REQUIRE(c.grad_rows || c.loss || (c.rows == 0 && c.reduction == 0), n + ": null loss");
  PTO_REQUIRE(!c.grad_rows || c.rows == 0 || (c.norm && c.z && (c.dh || c.dw)),
              n + ": null normalisers, target logits or gradients of a backward call");
  PTO_REQUIRE(!c.kd || c.vocab <= kMaxMarked, n + ": at most 393216 tokens");
  PTO_REQUIRE(c.grad_rows || c.reduction || !(c.dh || c.dw), n + ": gradients of losses per row need their gradients");
  PTO_REQUIRE((reinterpret_cast<uintptr_t>(c.w) & 15) == 0, n + ": weight must be 16-byte aligned");
  PTO_REQUIRE(ws || ws_bytes == 0, n + ": null workspace");
  return 0;
}

int run(const Call& c, int dtype, void* ws, size_t ws_bytes, void* stream) {
  if (check(c, dtype, ws, ws_bytes)) return -2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kBF16) return loss_t<bf16>(c, ws, ws_bytes, s);
  return few_rows(c) ? loss_t<float>(c, ws, ws_bytes, s) : loss_t<sp16>(c, ws, ws_bytes, s);
}

}  // namespace
}  // namespace pto

extern "C" {

size_t pto_linear_loss_workspace_bytes(int dtype, int64_t rows, int64_t d, int64_t vocab, int64_t k, int64_t ldw,
                                       double label_smoothing, int distillation, int backward, int dhidden, int dweight,
                                       int64_t chunk_bytes) {
  if (rows < 0 || d < 1 || vocab < 1 || k < 1) return 0;
  static const float one = 1.f;
  char some;
  pto::Call c{};
  c.rows = rows;
  c.d = d;
  c.vocab = vocab;
  c.k = k;
  c.ldw = ldw;
  c.smooth = label_smoothing;
  c.kd = distillation != 0;
  c.grad_rows = backward ? &one : nullptr;
  c.dh = dhidden ? &some : nullptr;
  c.dw = dweight ? &some : nullptr;
  c.chunk_bytes = chunk_bytes;
  switch (dtype) {
    case pto::kBF16: return pto::loss_ws_bytes<pto::bf16>(c);
    case pto::kF32: return pto::few_rows(c) ? pto::loss_ws_bytes<float>(c) : pto::loss_ws_bytes<pto::sp16>(c);
    default: return 0;
  }
}

int pto_linear_cross_entropy(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const int64_t* targets,
                             int dtype, int64_t rows, int64_t d, int64_t vocab, int64_t ignore_index,
                             double label_smoothing, double z_loss, int reduction, const float* grad_rows, float* loss,
                             float* norm, float* z, void* dhidden, void* dweight, int64_t chunk_bytes, void* workspace,
                             size_t ws_bytes, void* stream) {
  const pto::Call c{hidden, ldh,  weight,         ldw,    false, targets,   ignore_index, nullptr, nullptr, rows,    d,
                    vocab,  1,    1.0,            label_smoothing,   z_loss,       reduction, grad_rows, loss, norm,
                    z,      dhidden, dweight,     chunk_bytes, "linear_cross_entropy"};
  return pto::run(c, dtype, workspace, ws_bytes, stream);
}

int pto_linear_distillation(const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                            const float* teacher_logits, const int64_t* teacher_index, int dtype, int64_t rows,
                            int64_t d, int64_t vocab, int64_t k, double temperature, int reduction,
                            const float* grad_rows, float* loss, float* norm, float* z, void* dhidden, void* dweight,
                            int64_t chunk_bytes, void* workspace, size_t ws_bytes, void* stream) {
  const pto::Call c{hidden, ldh, weight, ldw, true, nullptr, 0,   teacher_logits, teacher_index, rows, d,
                    vocab,  k,   temperature, 0.0, 0.0, reduction, grad_rows, loss, norm,
                    z,      dhidden, dweight, chunk_bytes, "linear_distillation"};
  return pto::run(c, dtype, workspace, ws_bytes, stream);
}

int pto_scale_pair(void* x, int64_t n, void* y, int64_t m, int dtype, const float* factor, void* stream) {
  PTO_REQUIRE(dtype == pto::kF32 || dtype == pto::kBF16, "scale_pair: unsupported dtype code (fp32 and bf16)");
  PTO_REQUIRE(n >= 0 && m >= 0, "scale_pair: negative extent");
  PTO_REQUIRE((n == 0 || x) && (m == 0 || y) && (n + m == 0 || factor), "scale_pair: null operand");
  if (n + m == 0) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = (unsigned)std::min<int64_t>((std::max(n, m) + 2047) / 2048, 8 * pto::device_cus());
  if (dtype == pto::kBF16)
    hipLaunchKernelGGL(pto::scale_kernel<pto::bf16>, dim3(blocks), dim3(256), 0, s, static_cast<pto::bf16*>(x), n,
                       static_cast<pto::bf16*>(y), m, factor);
  else
    hipLaunchKernelGGL(pto::scale_kernel<float>, dim3(blocks), dim3(256), 0, s, static_cast<float*>(x), n,
                       static_cast<float*>(y), m, factor);
  PTO_LAUNCHED("scale_pair");
  return 0;
}

}  // extern "C"
