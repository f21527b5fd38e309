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
//   dots     z at the sparse targets, in fp32 (a dot product each);
//   logits   one MFMA product, whose epilogue takes the maximum and the sum of
//            exponentials of each row's 64 columns, and for gradients keeps the
//            block's logits in the workspace;
//   finish   joins a row's blocks to lse, gives its loss and turns the kept
//            logits into S;
//   dH, dW   two MFMA products (dW summed over the chunks in fp32).
// A pass over V·rows logits is 2·rows·d·V operations, the three products
// 6·rows·d·V: gradients found in the forward call need no second pass over the
// logits (8·rows·d·V). Where the rows' gradients come later (losses per row),
// lse and the targets' z are kept and the backward call forms S in the logits'
// epilogue.
#include <algorithm>
#include <cmath>

#include "aux_kernels.h"
#include "gemm_nt.h"

namespace pto {
namespace {

constexpr int kCols = 64;      // columns of a row that one entry of the statistics covers
constexpr int kMaxTeach = 1024;  // sparse targets per row
constexpr int64_t kChunkBytes = int64_t(2) << 30;  // kept logits of a chunk of rows
constexpr double kLn2 = 0.6931471805599453;

// bf16 inputs: a kept logit is how far it lies below its block's maximum, in
// log2, as a 16-bit fraction of 128 from the top. p is then off by at most
// 6.8e-4 (bf16's rounding of S: up to 3.9e-3) in the bytes that S takes in the
// end, and 0 stands for exponentials 2^-128 times the block's largest and
// less, which fp32 does not hold as normal numbers either. fp32 inputs keep
// fp32.
constexpr float kOctaves = 128.f;

// Sparse targets of a row, k per row in the caller's order. id: the token,
// -1 where there is none, -2 where it is outside the vocabulary; q: its share;
// put: what of S to take off at id (the first of equal ids has their sum, the
// others -1: nothing to do).
struct Targets {
  int* id;
  float *q, *put;
  float* entropy;  // per row: Σ q·log q
  int* kept;       // per row: whether the row counts
};

__global__ void __launch_bounds__(256) ce_targets_kernel(const int64_t* __restrict__ y, int64_t rows, int64_t vocab,
                                                         int64_t ignore, float share, Targets t,
                                                         float* __restrict__ loss) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= rows) return;
  const int64_t v = y[r];
  t.kept[r] = v != ignore;
  t.id[r] = v == ignore ? -1 : v >= 0 && v < vocab ? (int)v : -2;
  t.q[r] = t.put[r] = share;
  t.entropy[r] = 0.f;
  if (loss) loss[r] = 0.f;
}

__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One wave per row: the teacher's softmax over the entries that are there
// (id >= 0, logit above -inf).
__global__ void __launch_bounds__(256) kd_targets_kernel(const float* __restrict__ logit,
                                                         const int64_t* __restrict__ index, int64_t rows, int k,
                                                         int64_t vocab, float inv_temp, Targets t,
                                                         float* __restrict__ loss) {
  __shared__ int ids[4][kMaxTeach];
  __shared__ float qs[4][kMaxTeach];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t r = (int64_t)blockIdx.x * 4 + w;
  if (r >= rows) return;
  const float* lr = logit + r * k;
  const int64_t* ir = index + r * k;
  float m = -INFINITY;
  int n = 0;
  for (int e = lane; e < k; e += 64) {
    const float v = lr[e] * inv_temp;
    const int64_t id = ir[e];
    const bool there = id >= 0 && !(v == -INFINITY);
    ids[w][e] = !there ? -1 : id < vocab ? (int)id : -2;
    qs[w][e] = v;
    if (there) {
      m = fmaxf(m, v);
      ++n;
    }
  }
  m = wave_max(m);
  n = __any(n > 0);
  float s = 0.f;
  for (int e = lane; e < k; e += 64)
    if (ids[w][e] != -1) s += expf(qs[w][e] - m);
  s = wave_sum(s);
  const float logs = logf(s);
  float ent = 0.f;
  for (int e = lane; e < k; e += 64) {
    float q = 0.f;
    if (ids[w][e] != -1) {
      const float logq = qs[w][e] - m - logs;
      q = expf(logq);
      if (q != 0.f) ent += q * logq;
    }
    qs[w][e] = q;
  }
  ent = wave_sum(ent);
  __builtin_amdgcn_s_waitcnt(PTO_LGKM0);
  __builtin_amdgcn_wave_barrier();
  for (int e = lane; e < k; e += 64) {
    const int id = ids[w][e];
    float put = -1.f;
    if (id >= 0) {
      put = 0.f;
      for (int o = 0; o < k; ++o) {
        if (ids[w][o] != id) continue;
        if (o < e) {
          put = -1.f;
          break;
        }
        put += qs[w][o];
      }
    }
    t.id[r * k + e] = id;
    t.q[r * k + e] = qs[w][e];
    t.put[r * k + e] = put;
  }
  if (lane == 0) {
    t.kept[r] = n;
    t.entropy[r] = ent;
    if (loss) loss[r] = 0.f;
  }
}

// list = the rows that count in order, then the others; count[0] = how many
// count. One workgroup, each thread a run of rows.
__global__ void __launch_bounds__(1024) list_rows_kernel(const int* __restrict__ kept, int64_t rows,
                                                         int* __restrict__ list, int* __restrict__ count) {
  __shared__ int part[1024];
  const int t = threadIdx.x;
  const int64_t per = (rows + 1023) / 1024, r0 = min(rows, t * per), r1 = min(rows, r0 + per);
  int n = 0;
  for (int64_t r = r0; r < r1; ++r) n += kept[r] != 0;
  part[t] = n;
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    const int add = t >= o ? part[t - o] : 0;
    __syncthreads();
    part[t] += add;
    __syncthreads();
  }
  const int total = part[1023];
  int yes = part[t] - n;
  int64_t no = total + r0 - yes;
  for (int64_t r = r0; r < r1; ++r) {
    if (kept[r] != 0)
      list[yes++] = (int)r;
    else
      list[no++] = (int)r;
  }
  if (t == 0) count[0] = total;
}

// The rows of a chunk, as the kernels see them.
struct Chunk {
  const int* list;
  const int* count;
  int64_t rows;  // of the call
  int base, cap;  // first listed row, most rows
  __device__ __forceinline__ int live() const { return max(0, min(cap, count[0] - base)); }
  // rows that products reading them along K see: zero rows up to a multiple of kPadK
  __device__ __forceinline__ int padded() const { return (live() + kPadK - 1) / kPadK * kPadK; }
};

// A row of n elements (any alignment) into a padded one, one wave.
template <typename T>
__device__ __forceinline__ void copy_row(const T* __restrict__ src, int64_t n, T* __restrict__ dst, int64_t ld,
                                         int lane) {
  constexpr int E = 16 / (int)sizeof(T);
  for (int64_t c = lane * E; c < ld; c += 64 * E) {
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

template <typename T>
__global__ void __launch_bounds__(256) gather_kernel(Chunk ch, const T* __restrict__ h, int64_t ldh, int64_t d,
                                                     T* __restrict__ hc, int64_t ldc, T* __restrict__ dh) {
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= ch.padded() && (dh == nullptr || ch.base + i >= ch.rows || i >= ch.cap)) return;
  if (i < ch.live()) {
    copy_row(h + ch.list[ch.base + i] * ldh, d, hc + i * ldc, ldc, lane);
    return;
  }
  constexpr int E = 16 / (int)sizeof(T);
  if (i < ch.padded())
    for (int64_t c = lane * E; c < ldc; c += 64 * E) *reinterpret_cast<uint4*>(hc + i * ldc + c) = make_uint4(0, 0, 0, 0);
  if (dh && i < ch.cap && ch.base + i < ch.rows) {
    T* row = dh + ch.list[ch.base + i] * d;
    for (int64_t c = lane; c < d; c += 64) row[c] = T(0.f);
  }
}

// W padded to a multiple of kPadK rows and columns.
template <typename T>
__global__ void __launch_bounds__(256) pad_weight_kernel(const T* __restrict__ w, int64_t ldw, int64_t vocab, int64_t d,
                                                         T* __restrict__ out, int64_t ldo, int64_t rows) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  copy_row(w + min(r, vocab - 1) * ldw, r < vocab ? d : 0, out + r * ldo, ldo, threadIdx.x & 63);
}

// z at the sparse targets in units of log2 (scale = log2(e)/T), one wave each:
// out[(base + i)·k + e].
template <typename T>
__global__ void __launch_bounds__(256) dots_kernel(Chunk ch, const T* __restrict__ hc, int64_t ldc,
                                                   const T* __restrict__ w, int64_t ldw, int64_t d, int k, Targets t,
                                                   float scale, float* __restrict__ out) {
  constexpr int E = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t i = id / k, e = id % k;
  if (i >= ch.live()) return;
  const int v = t.id[(int64_t)ch.list[ch.base + i] * k + e];
  float s = v == -2 ? NAN : 0.f;
  if (v >= 0) {
    const T* hr = hc + i * ldc;
    const T* wr = w + v * ldw;
    for (int64_t c = lane * E; c < d; c += 64 * E) {
      const uint4 a = *reinterpret_cast<const uint4*>(hr + c);
      const T* x = reinterpret_cast<const T*>(&a);
      if (c + E <= d) {
        const uint4 b = ld16(wr + c);
        const T* y = reinterpret_cast<const T*>(&b);
#pragma unroll
        for (int q = 0; q < E; ++q) s = fmaf(to_f(x[q]), to_f(y[q]), s);
      } else {
        for (int q = 0; q < E; ++q)
          if (c + q < d) s = fmaf(to_f(x[q]), to_f(wr[c + q]), s);
      }
    }
    s = wave_sum(s) * scale;
  }
  if (lane == 0) out[(ch.base + i) * k + e] = s;
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

// What a row's slopes need besides its logits: S = pa·2^(t − lse2) + pu.
struct RowSlope {
  float lse2, pa, pu;
};

// Epilogue of the logits' product, from the accumulators (kDirect): 16 lanes
// have a row's 64 columns, four each. Through LDS staging in runs of eight the
// same work took 14 us of a 256² tile's 69 at d = 2048, most of it VALU.
template <typename T, bool KEEP, bool SLOPE>
struct EpiLogits {
  typedef float S;
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
  __device__ __forceinline__ bool adjust(GemmArgs& g, int, int row0, int) const {
    g.M = SLOPE ? ch.padded() : ch.live();
    return row0 < g.M;
  }
  __device__ __forceinline__ int q_rows() const { return vocab; }
  __device__ __forceinline__ void finish(int) const {}
  template <class V, int FM, int FN>
  __device__ __forceinline__ void direct(const V (&acc)[FM][FN], char* lds, const GemmArgs& g, int wr0, int wc0,
                                         int lane) const {
    if (wc0 >= g.N || wr0 >= g.M) return;
    const int l = lane & 15, sub = (lane >> 4) * 4, c0 = wc0 + 4 * l;
    const bool whole = wc0 + kCols <= vocab;  // false in the last block of a row at most
    RowSlope* const rs = reinterpret_cast<RowSlope*>(lds);
    if (SLOPE) {
      for (int r = lane; r < FM * 16; r += 64)
        if (wr0 + r < g.M) rs[r] = row[wr0 + r];
      __builtin_amdgcn_s_waitcnt(PTO_LGKM0);
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wr0 + fm * 16 + sub + r;
        const bool live = i < g.M;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = acc[fm][k][r];
        if (SLOPE) {
          const RowSlope p = rs[fm * 16 + sub + r];
          float t[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) t[k] = fmaf(p.pa, pow2(fmaf(v[k], scale, -p.lse2)), p.pu);
          if (!whole) {
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = c0 + k < vocab ? t[k] : 0.f;
          }
          if (live) st4(static_cast<T*>(kept) + i * ld + c0, t);
          continue;
        }
        if (!whole) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = c0 + k < vocab ? v[k] : -INFINITY;
        }
        const float m = max16(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
        const float ref = m == -INFINITY ? 0.f : m * scale;  // a block of nothing but -inf sums to 0
        float x[4], s = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = fmaf(v[k], scale, -ref);
          s += pow2(x[k]);
        }
        s = sum16(s);
        if (live && l == 0) stats[i * blocks + wc0 / kCols] = make_float2(ref, s);
        if (sums) {
          float z = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) z += c0 + k < vocab ? v[k] : 0.f;
          z = sum16(z) * scale;
          if (live && l == 0) sums[i * blocks + wc0 / kCols] = z;
        }
        if (KEEP && live) {
          if constexpr (sizeof(T) == 2) {
            uint2 u;
            u.x = encode(x[0], x[1]);
            u.y = encode(x[2], x[3]);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(kept) + i * ld + c0) = u;
          } else {
            float t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = v[k] * scale;
            st4(static_cast<float*>(kept) + i * ld + c0, t);
          }
        }
      }
    }
  }
  // (x/128 + 1)·65535, rounded, between 0 and 65535
  __device__ __forceinline__ static unsigned encode(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(fmaf(a, 1.f / kOctaves, 1.f),
                                                                        fmaf(b, 1.f / kOctaves, 1.f)));
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
  float inv_temp;
  int k;
  int reduction;  // 0: gradients (if any) under grad_rows, 1: mean, 2: sum
};

// a and f of a row (see the top), as the slope of exp2(t - lse2) and the constant.
__device__ __forceinline__ RowSlope row_slope(const LossSpec& sp, float lse2, float g) {
  RowSlope r;
  r.lse2 = lse2;
  const float a = g * sp.lambda * sp.inv_temp;
  r.pa = a * (1.f + 2.f * sp.zeta * (float)(kLn2 * lse2));
  // where the logits overflow nothing of the row is left standing as a number
  if (!(fabsf(lse2) < INFINITY)) r.pa = NAN;
  r.pu = -a * sp.smooth;
  return r;
}

// S at a row's sparse targets, after the dense part was written.
template <typename T>
__device__ __forceinline__ void put_targets(T* srow, const RowSlope& rs, const LossSpec& sp, float g, const int* id,
                                            const float* put, const float* z, int first, int step) {
  const float a = g * sp.lambda * sp.inv_temp;
  for (int e = first; e < sp.k; e += step)
    if (id[e] >= 0 && put[e] >= 0.f) srow[id[e]] = T(fmaf(rs.pa, pow2(z[e] - rs.lse2), fmaf(-a, put[e], rs.pu)));
}

// One workgroup per listed row: lse, the loss and (S not null) S in place of
// the kept logits. losses is per row of the call, lse2_out per listed row.
template <typename T, bool SLOPES>
__global__ void __launch_bounds__(256) finish_kernel(Chunk ch, const float2* __restrict__ stats,
                                                     const float* __restrict__ sums, int64_t blocks, LossSpec sp,
                                                     Targets tg, const float* __restrict__ z, int vocab,
                                                     void* __restrict__ kept, int64_t ld, float* __restrict__ losses,
                                                     float* __restrict__ lse2_out) {
  const int i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int live = ch.live();
  constexpr int E = 16 / (int)sizeof(T);
  if (i >= live) {
    if (SLOPES && i < ch.padded())
      for (int64_t c = tid * E; c < ld; c += 256 * E)
        *reinterpret_cast<uint4*>(static_cast<T*>(kept) + i * ld + c) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int row = ch.list[ch.base + i];
  const float2* st = stats + i * blocks;
  const int* id = tg.id + (int64_t)row * sp.k;
  const float* q = tg.q + (int64_t)row * sp.k;
  const float* zr = z + (int64_t)(ch.base + i) * sp.k;
  __shared__ float red[4][4];
  float m = -INFINITY;
  for (int64_t c = tid; c < blocks; c += 256)
    if (st[c].y != 0.f) m = fmaxf(m, st[c].x);
  m = wave_max(m);
  if (lane == 0) red[0][w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  if (m == -INFINITY) m = 0.f;
  float s = 0.f, sz = 0.f, qz = 0.f;
  for (int64_t c = tid; c < blocks; c += 256) {
    s += st[c].y == 0.f ? 0.f : st[c].y * pow2(st[c].x - m);
    if (sums) sz += sums[i * blocks + c];
  }
  for (int e = tid; e < sp.k; e += 256)
    if (id[e] != -1) qz += q[e] * zr[e];
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
  const float lse2 = m + log2f(s);
  if (tid == 0) {
    const double lse = kLn2 * ((double)m + (double)log2f(s));
    const double nat = lse - kLn2 * ((double)qz + (double)sp.smooth * sz) + tg.entropy[row];
    losses[row] = (float)(sp.lambda * nat + (double)sp.zeta * lse * lse);
    if (lse2_out) lse2_out[ch.base + i] = lse2;
  }
  if constexpr (SLOPES) {
    const float g = sp.reduction == 1 ? 1.f / (float)ch.count[0] : 1.f;
    RowSlope rs = row_slope(sp, lse2, g);
    if (!(fabsf(qz) < INFINITY)) rs.pa = NAN;  // a target outside the vocabulary, or one that is not a number
    for (int64_t c = tid * E; c < ld; c += 256 * E) {
      float o[E];
      if constexpr (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<uint16_t*>(kept) + i * ld + c);
        const unsigned uw[4] = {u.x, u.y, u.z, u.w};
        const float off = st[c / kCols].x - rs.lse2 - kOctaves;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const unsigned x = e & 1 ? uw[e / 2] >> 16 : uw[e / 2] & 0xffffu;
          const float p = x ? pow2(fmaf((float)x, kOctaves / 65535.f, off)) : 0.f;
          o[e] = c + e < vocab ? fmaf(rs.pa, p, rs.pu) : 0.f;
        }
        uint4 r;
        T* re = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int e = 0; e < E; ++e) re[e] = T(o[e]);
        *reinterpret_cast<uint4*>(static_cast<T*>(kept) + i * ld + c) = r;
      } else {
        float* p = static_cast<float*>(kept) + i * ld + c;
        const float4 x = *reinterpret_cast<const float4*>(p);
        const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = c + e < vocab ? fmaf(rs.pa, pow2(xs[e] - rs.lse2), rs.pu) : 0.f;
        *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
      }
    }
    __syncthreads();  // the dense part is written before the targets' entries replace theirs
    put_targets(static_cast<T*>(kept) + i * ld, rs, sp, g, id, tg.put + (int64_t)row * sp.k, zr, tid, 256);
  }
}

// Gradients of losses per row: what the logits' epilogue needs of each row
// (zero for the pad rows).
__global__ void __launch_bounds__(256) row_slopes_kernel(Chunk ch, LossSpec sp, Targets tg, const float* __restrict__ z,
                                                         const float* __restrict__ lse2,
                                                         const float* __restrict__ grad_rows, RowSlope* out) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= ch.padded()) return;
  RowSlope rs{0.f, 0.f, 0.f};
  if (i < ch.live()) {
    const int64_t at = ch.base + i, row = ch.list[at];
    rs = row_slope(sp, lse2[at], grad_rows[row]);
    for (int e = 0; e < sp.k; ++e)
      if (tg.id[row * sp.k + e] != -1 && !(fabsf(tg.q[row * sp.k + e] * z[at * sp.k + e]) < INFINITY)) rs.pa = NAN;
  }
  out[i] = rs;
}
template <typename T>
__global__ void __launch_bounds__(64) put_targets_kernel(Chunk ch, LossSpec sp, Targets tg, const float* __restrict__ z,
                                                         const RowSlope* __restrict__ rows,
                                                         const float* __restrict__ grad_rows, T* __restrict__ s,
                                                         int64_t ld) {
  const int i = blockIdx.x;
  if (i >= ch.live()) return;
  const int64_t at = ch.base + i, row = ch.list[at];
  put_targets(s + i * ld, rows[i], sp, grad_rows[row], tg.id + row * sp.k, tg.put + row * sp.k, z + at * sp.k,
              threadIdx.x, 64);
}

// The loss of the call: a sum in a fixed order, over the count for the mean
// (no row counts: 0).
__global__ void __launch_bounds__(1024) reduce_loss_kernel(const float* __restrict__ losses, int64_t rows,
                                                           const int* __restrict__ count, int mean,
                                                           float* __restrict__ out) {
  __shared__ double red[1024];
  double s = 0;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) s += losses[r];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 512; w > 0; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[0] = (float)(red[0] / (mean ? max(1, count[0]) : 1));
}

// ------------------------------------------------------------ gradients

// dH: rows of the chunk to their places.
template <typename T>
struct EpiRows {
  typedef float S;
  Chunk ch;
  T* dst;
  int64_t ld;
  typedef NoPre Pre;
  typedef NoPre PreT;
  static constexpr bool kVoIsV = true;
  __device__ __forceinline__ bool has_t() const { return false; }
  __device__ __forceinline__ bool adjust(GemmArgs& g, int, int row0, int) const {
    g.M = ch.live();
    return row0 < g.M;
  }
  __device__ __forceinline__ void load(int, int, int, int, int, Pre&) const {}
  __device__ __forceinline__ void load_t(int, int, int, int, PreT&) const {}
  __device__ __forceinline__ void put_t(int, int, int, const S*, int, const PreT&) const {}
  __device__ __forceinline__ void finish(int) const {}
  __device__ __forceinline__ void put(int, int i, int j0, const S* v, int kbeg, int n, const Pre&, S*) const {
    st8<T, S>(dst + ch.list[ch.base + i] * ld + j0, v, kbeg, n);
  }
};

// dH of few rows: the vocabulary split over the batch index, partial sums to
// the workspace.
struct EpiPart {
  typedef float S;
  Chunk ch;
  float* dst;
  int64_t ld, sd;
  int len, total;  // K of a slice, of all
  typedef NoPre Pre;
  typedef NoPre PreT;
  static constexpr bool kVoIsV = true;
  __device__ __forceinline__ bool has_t() const { return false; }
  __device__ __forceinline__ bool adjust(GemmArgs& g, int b, int row0, int) const {
    g.M = ch.live();
    g.K = max(0, min(len, total - b * len));
    return row0 < g.M;
  }
  __device__ __forceinline__ void load(int, int, int, int, int, Pre&) const {}
  __device__ __forceinline__ void load_t(int, int, int, int, PreT&) const {}
  __device__ __forceinline__ void put_t(int, int, int, const S*, int, const PreT&) const {}
  __device__ __forceinline__ void finish(int) const {}
  __device__ __forceinline__ void put(int b, int i, int j0, const S* v, int kbeg, int n, const Pre&, S*) const {
    st8<float, S>(dst + b * sd + i * ld + j0, v, kbeg, n);
  }
};
template <typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(Chunk ch, const float* __restrict__ part, int64_t ld,
                                                         int64_t sd, int parts, int64_t d, T* __restrict__ dst) {
  const int i = blockIdx.x;
  if (i >= ch.live()) return;
  T* row = dst + ch.list[ch.base + i] * d;
  for (int64_t c = threadIdx.x; c < d; c += 256) {
    float s = 0.f;
    for (int p = 0; p < parts; ++p) s += part[p * sd + i * ld + c];
    row[c] = convert<T>(s);
  }
}

// dW over the chunks of rows: acc = v (first), acc + v, and out = acc + v
// rounded (last); acc is out where the chunk is the only one or out is fp32.
template <typename T>
struct EpiWeight {
  typedef float S;
  Chunk ch;
  float* acc;
  T* out;
  int64_t ld;
  int first, last;
  typedef Raw8<float> Pre;
  typedef NoPre PreT;
  static constexpr bool kVoIsV = true;
  __device__ __forceinline__ bool has_t() const { return false; }
  __device__ __forceinline__ bool adjust(GemmArgs& g, int, int, int) const {
    g.K = ch.padded();
    return g.K > 0 || first || last;
  }
  __device__ __forceinline__ void load(int, int i, int j0, int kbeg, int n, Pre& p) const {
    if (!first) ld8_pre<float>(acc + i * ld + j0, p, kbeg, n);
  }
  __device__ __forceinline__ void load_t(int, int, int, int, PreT&) const {}
  __device__ __forceinline__ void put_t(int, int, int, const S*, int, const PreT&) const {}
  __device__ __forceinline__ void finish(int) const {}
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
    if (last)
      st8<T, float>(out + i * ld + j0, r, kbeg, n);
    else
      st8<float, float>(acc + i * ld + j0, r, kbeg, n);
  }
};

// x *= s[0] in place, nothing where s[0] is 1 (the gradient of a loss that is
// itself differentiated).
template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(T* __restrict__ x, int64_t n, const float* __restrict__ s) {
  const float f = s[0];
  if (f == 1.f) return;
  constexpr int E = 16 / (int)sizeof(T);
  const int64_t step = (int64_t)gridDim.x * 256 * E;
  for (int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * E; c < n; c += step) {
    if (c + E <= n) {
      uint4 u = ld16(x + c);
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int k = 0; k < E; ++k) e[k] = convert<T>(to_f(e[k]) * f);
      st16(x + c, u);
    } else {
      for (int64_t k = c; k < n; ++k) x[k] = convert<T>(to_f(x[k]) * f);
    }
  }
}

// ------------------------------------------------------------ host

struct Call {
  const void* h;
  int64_t ldh;
  const void* w;
  int64_t ldw;
  const int64_t* y;       // cross entropy
  int64_t ignore;
  const float* teacher;   // distillation
  const int64_t* index;
  int64_t rows, d, vocab, k;
  double temp, smooth, zeta;
  int reduction;
  const float* grad_rows;
  float *loss, *lse, *z;
  void *dh, *dw;
  int64_t chunk_bytes;
  const char* name;
};

// Parts of the vocabulary that dH of a chunk is split into: as many as leave
// no CU idle through a long loop over K, each at least kPadK deep; the partial
// sums (8 bytes of traffic an element) count against it.
template <typename T>
int grad_parts(int64_t rows, int64_t d, int64_t vp, int* tile) {
  typedef typename TileSet<T>::big Big;
  typedef typename TileSet<T>::small Small;
  const int64_t cus = device_cus(), units = vp / kPadK;
  // microseconds of one unit of K on one CU, per element of a tile
  const double us = sizeof(T) == 2 ? 3.6 / 65536 : 5.0 / 16384;
  double best = 0;
  int parts = 1;
  for (int big = 0; big < 2; ++big) {
    const int64_t bm = big ? Big::BM : Small::BM, bn = big ? Big::BN : Small::BN;
    const int64_t tiles = ((rows + bm - 1) / bm) * ((d + bn - 1) / bn);
    for (int p = 1; p <= 64 && p <= units; p *= 2) {
      const double unit = bm * bn * us * (big ? 1.0 : TileSet<T>::kBigRate);
      double t = double((tiles * p + cus - 1) / cus) * ((units + p - 1) / p) * unit;
      if (p > 1) t += 5 + p * (double)rows * d * 8 / 4e6;
      if ((!big && p == 1) || t < best) {
        best = t;
        parts = p;
        *tile = big;
      }
    }
  }
  return parts;
}

template <typename T>
struct Ws {
  int64_t dp, vp, blocks, cap, capp;
  bool pad_w;
  int parts, part_tile = 0;
  Targets t;
  int *list, *count;
  T *hc, *wp;
  float2* stats;
  float *sums, *losses, *lse, *z;
  RowSlope* slopes;
  void* kept;
  T *keptT, *hcT, *wT;
  float *part, *acc;
  int64_t chunks(const Call& c) const { return c.rows ? (c.rows + cap - 1) / cap : 0; }
  Ws(Carver& cv, const Call& c) {
    const bool f32 = sizeof(T) == 4, grads = c.dh || c.dw;
    dp = round_up(c.d, kPadK);
    vp = round_up(c.vocab, kPadK);
    blocks = vp / kCols;
    const int64_t per = grads ? vp * (int64_t)sizeof(T) * (f32 && c.dw ? 2 : 1) : blocks * 8;
    cap = (c.chunk_bytes > 0 ? c.chunk_bytes : kChunkBytes) / per;
    cap = std::min(std::max<int64_t>(cap / 256 * 256, 256), std::max<int64_t>(c.rows, 1));
    capp = round_up(cap, kPadK);
    pad_w = c.d % kPadK || c.ldw % (16 / sizeof(T)) || (!f32 && c.dh && c.vocab % kPadK);
    t.id = cv.take<int>(c.rows * c.k);
    t.q = cv.take<float>(c.rows * c.k);
    t.put = cv.take<float>(c.rows * c.k);
    t.entropy = cv.take<float>(c.rows);
    t.kept = cv.take<int>(c.rows);
    list = cv.take<int>(c.rows);
    count = cv.take<int>(4);
    hc = cv.take<T>(capp * dp);
    wp = pad_w ? cv.take<T>(vp * dp) : nullptr;
    losses = cv.take<float>(c.rows);
    lse = cv.take<float>(c.rows);
    z = cv.take<float>(c.rows * c.k);
    stats = c.grad_rows ? nullptr : cv.take<float2>(cap * blocks);
    sums = c.smooth != 0 && !c.grad_rows ? cv.take<float>(cap * blocks) : nullptr;
    slopes = c.grad_rows ? cv.take<RowSlope>(capp) : nullptr;
    kept = grads ? static_cast<void*>(cv.take<T>(capp * vp)) : nullptr;
    keptT = f32 && c.dw ? cv.take<T>(c.vocab * capp) : nullptr;
    hcT = f32 && c.dw ? cv.take<T>(c.d * capp) : nullptr;
    wT = f32 && c.dh ? cv.take<T>(c.d * vp) : nullptr;
    parts = c.dh ? grad_parts<T>(cap, c.d, vp, &part_tile) : 1;
    part = parts > 1 ? cv.take<float>(parts * cap * dp) : nullptr;
    acc = !f32 && c.dw && chunks(c) > 1 ? cv.take<float>(c.vocab * c.d) : nullptr;
  }
};

template <typename T>
size_t loss_ws_bytes(const Call& c) {
  Carver cv(nullptr, 0);
  Ws<T> w(cv, c);
  return cv.used + 512;
}

// A product with the tile given (K-contiguous operands).
template <typename T, class Epi>
int launch_nt(const GemmArgs& g, const Epi& e, int batch, bool big, hipStream_t s, const char* name) {
  PTO_REQUIRE(g.K % ring_k<T>() == 0 && g.ldp % (16 / sizeof(T)) == 0 && g.ldq % (16 / sizeof(T)) == 0 &&
                  ((reinterpret_cast<uintptr_t>(g.P) | reinterpret_cast<uintptr_t>(g.Q)) & 15) == 0,
              std::string(name) + ": operands not padded or not 16-byte aligned");
  // a direct epilogue needs 64-column wave tiles: fp32's 128² tile, either bf16 tile
  if (big || (IsDirect<Epi>::value && sizeof(T) == 4))
    return launch_gemm_cfg<T, typename TileSet<T>::big, false>(g, e, batch, s, name);
  if constexpr (!IsDirect<Epi>::value || sizeof(T) == 2) return launch_gemm_cfg<T, typename TileSet<T>::small, false>(g, e, batch, s, name);
  return -1;
}

template <typename T>
int loss_t(const Call& c, void* ws, size_t ws_bytes, hipStream_t s) {
  constexpr bool f32 = sizeof(T) == 4;
  Carver cv(ws, ws_bytes);
  const Ws<T> w(cv, c);
  PTO_REQUIRE(!cv.overflow, std::string(c.name) + ": workspace too small");
  const bool grads = c.dh || c.dw;
  const T* W = static_cast<const T*>(c.w);
  int64_t ldw = c.ldw;
  if (c.rows == 0) {  // no row: loss and gradients of nothing
    if (c.reduction && c.loss) {
      hipLaunchKernelGGL(reduce_loss_kernel, dim3(1), dim3(1024), 0, s, w.losses, 0, w.count, 0, c.loss);
      PTO_LAUNCHED("reduce_loss");
    }
  } else {
    float* losses = c.reduction || !c.loss ? w.losses : c.loss;
    if (c.y) {
      hipLaunchKernelGGL(ce_targets_kernel, dim3((unsigned)((c.rows + 255) / 256)), dim3(256), 0, s, c.y, c.rows,
                         c.vocab, c.ignore, (float)(1.0 - c.smooth), w.t, losses);
    } else {
      hipLaunchKernelGGL(kd_targets_kernel, dim3((unsigned)((c.rows + 3) / 4)), dim3(256), 0, s, c.teacher, c.index,
                         c.rows, (int)c.k, c.vocab, (float)(1.0 / c.temp), w.t, losses);
    }
    PTO_LAUNCHED("loss_targets");
    hipLaunchKernelGGL(list_rows_kernel, dim3(1), dim3(1024), 0, s, w.t.kept, c.rows, w.list, w.count);
    PTO_LAUNCHED("list_rows");
  }
  if (w.pad_w) {
    hipLaunchKernelGGL(pad_weight_kernel<T>, dim3((unsigned)((w.vp + 3) / 4)), dim3(256), 0, s, W, ldw, c.vocab, c.d,
                       w.wp, w.dp, w.vp);
    PTO_LAUNCHED("pad_weight");
    W = w.wp;
    ldw = w.dp;
  }
  if constexpr (f32) {
    if (c.dh && launch_pack<T, T, float>(W, c.vocab, c.d, ldw, 0, nullptr, nullptr, 0, 0, w.wT, w.vp, 0, false, 1, s))
      return -1;
  }
  float* lse = c.lse ? c.lse : w.lse;
  float* z = c.z ? c.z : w.z;
  const float scale = (float)(1.4426950408889634 / c.temp);
  const LossSpec sp{(float)(c.temp * c.temp), (float)(c.smooth / c.vocab), (float)c.zeta, (float)(1.0 / c.temp),
                    (int)c.k, c.reduction};
  const int64_t chunks = std::max<int64_t>(w.chunks(c), c.dw ? 1 : 0);  // no rows: dW is still written
  for (int64_t n = 0; n < chunks; ++n) {
    const Chunk ch{w.list, w.count, c.rows, (int)(n * w.cap), (int)std::min(w.cap, c.rows - n * w.cap)};
    const int capp = (int)round_up(ch.cap, kPadK);
    if (c.rows > 0) {
      hipLaunchKernelGGL(gather_kernel<T>, dim3((unsigned)(capp / 4)), dim3(256), 0, s, ch, static_cast<const T*>(c.h),
                         c.ldh, c.d, w.hc, w.dp, static_cast<T*>(c.dh));
      PTO_LAUNCHED("gather");
      GemmArgs g{w.hc, w.dp, 0, W, ldw, 0, ch.cap, (int)w.vp, (int)w.dp, 0, 0, nullptr};
      const bool big = pick_tile<T, false>(ch.cap, w.vp, 1) == 1;
      if (c.grad_rows) {
        hipLaunchKernelGGL(row_slopes_kernel, dim3((unsigned)((capp + 255) / 256)), dim3(256), 0, s, ch, sp, w.t, z,
                           lse, c.grad_rows, w.slopes);
        PTO_LAUNCHED("row_slopes");
        g.M = capp;
        const EpiLogits<T, false, true> e{ch, (int)c.vocab, scale, nullptr, nullptr, w.blocks, w.kept, w.vp, w.slopes};
        if (launch_nt<T>(g, e, 1, big, s, "loss_logits")) return -1;
        hipLaunchKernelGGL(put_targets_kernel<T>, dim3((unsigned)ch.cap), dim3(64), 0, s, ch, sp, w.t, z, w.slopes,
                           c.grad_rows, static_cast<T*>(w.kept), w.vp);
        PTO_LAUNCHED("put_targets");
      } else {
        hipLaunchKernelGGL(dots_kernel<T>, dim3((unsigned)((ch.cap * c.k + 3) / 4)), dim3(256), 0, s, ch, w.hc, w.dp,
                           static_cast<const T*>(c.w), c.ldw, c.d, (int)c.k, w.t, scale, z);
        PTO_LAUNCHED("dots");
        float* losses = c.reduction ? w.losses : c.loss;
        if (grads) {
          const EpiLogits<T, true, false> e{ch, (int)c.vocab, scale, w.stats, w.sums, w.blocks, w.kept, w.vp, nullptr};
          if (launch_nt<T>(g, e, 1, big, s, "loss_logits")) return -1;
          hipLaunchKernelGGL((finish_kernel<T, true>), dim3((unsigned)capp), dim3(256), 0, s, ch, w.stats, w.sums,
                             w.blocks, sp, w.t, z, (int)c.vocab, w.kept, w.vp, losses, lse);
        } else {
          const EpiLogits<T, false, false> e{ch,       (int)c.vocab, scale,   w.stats, w.sums,
                                             w.blocks, nullptr,      w.vp,    nullptr};
          if (launch_nt<T>(g, e, 1, big, s, "loss_logits")) return -1;
          hipLaunchKernelGGL((finish_kernel<T, false>), dim3((unsigned)ch.cap), dim3(256), 0, s, ch, w.stats, w.sums,
                             w.blocks, sp, w.t, z, (int)c.vocab, nullptr, w.vp, losses, lse);
        }
        PTO_LAUNCHED("finish");
      }
    }
    const T* S = static_cast<const T*>(w.kept);
    if (c.dh && c.rows > 0) {
      const int len = (int)(round_up((w.vp / kPadK + w.parts - 1) / w.parts, 1) * kPadK);
      GemmArgs g{S, w.vp, 0, f32 ? w.wT : W, f32 ? w.vp : ldw, 0, ch.cap, (int)c.d, (int)w.vp, 0, 0, nullptr};
      if (w.parts > 1) {
        g.K = len;
        g.sP = len;
        g.sQ = f32 ? len : len * ldw;
        const EpiPart e{ch, w.part, w.dp, w.cap * w.dp, len, (int)w.vp};
        if constexpr (f32) {
          if (launch_nt<T>(g, e, w.parts, w.part_tile, s, "loss_dhidden")) return -1;
        } else {
          if (launch_gemm_qn(g, e, w.parts, s, "loss_dhidden", w.part_tile)) return -1;
        }
        hipLaunchKernelGGL(join_parts_kernel<T>, dim3((unsigned)ch.cap), dim3(256), 0, s, ch, w.part, w.dp,
                           w.cap * w.dp, w.parts, c.d, static_cast<T*>(c.dh));
        PTO_LAUNCHED("join_parts");
      } else {
        const EpiRows<T> e{ch, static_cast<T*>(c.dh), c.d};
        if constexpr (f32) {
          if (launch_nt<T>(g, e, 1, w.part_tile, s, "loss_dhidden")) return -1;
        } else {
          if (launch_gemm_qn(g, e, 1, s, "loss_dhidden", w.part_tile)) return -1;
        }
      }
    }
    if (c.dw) {
      const bool first = n == 0, last = n == chunks - 1;
      T* dw = static_cast<T*>(c.dw);
      if constexpr (f32) {
        if (launch_pack<T, T, float>(S, capp, c.vocab, w.vp, 0, nullptr, nullptr, 0, 0, w.keptT, w.capp, 0, false, 1,
                                     s) ||
            launch_pack<T, T, float>(w.hc, capp, c.d, w.dp, 0, nullptr, nullptr, 0, 0, w.hcT, w.capp, 0, false, 1, s))
          return -1;
        const GemmArgs g{w.keptT, w.capp, 0, w.hcT, w.capp, 0, (int)c.vocab, (int)c.d, capp, 0, 0, nullptr};
        const EpiWeight<T> e{ch, dw, dw, c.d, first, last};
        if (launch_nt<T>(g, e, 1, pick_tile<T, false>(c.vocab, c.d, 1) == 1, s, "loss_dweight")) return -1;
      } else {
        const GemmArgs g{S, w.vp, 0, w.hc, w.dp, 0, (int)c.vocab, (int)c.d, capp, 0, 0, nullptr};
        const EpiWeight<T> e{ch, w.acc, dw, c.d, first, last};
        if (launch_gemm_qn<EpiWeight<T>, true>(g, e, 1, s, "loss_dweight")) return -1;
      }
    }
  }
  if (c.rows > 0 && c.reduction && c.loss) {
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
  PTO_REQUIRE(!c.grad_rows || c.rows == 0 || (c.lse && c.z && (c.dh || c.dw)),
              n + ": null lse, target logits or gradients of a backward call");
  PTO_REQUIRE(c.grad_rows || c.reduction || !(c.dh || c.dw), n + ": gradients of losses per row need their gradients");
  PTO_REQUIRE((reinterpret_cast<uintptr_t>(c.w) & 15) == 0, n + ": weight must be 16-byte aligned");
  PTO_REQUIRE(ws || ws_bytes == 0, n + ": null workspace");
  return 0;
}

int run(const Call& c, int dtype, void* ws, size_t ws_bytes, void* stream) {
  if (check(c, dtype, ws, ws_bytes)) return -2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == kBF16 ? loss_t<bf16>(c, ws, ws_bytes, s) : loss_t<float>(c, ws, ws_bytes, s);
}

}  // namespace
}  // namespace pto

extern "C" {

size_t pto_linear_loss_workspace_bytes(int dtype, int64_t rows, int64_t d, int64_t vocab, int64_t k, int64_t ldw,
                                       double label_smoothing, int backward, int dhidden, int dweight,
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
  c.grad_rows = backward ? &one : nullptr;
  c.dh = dhidden ? &some : nullptr;
  c.dw = dweight ? &some : nullptr;
  c.chunk_bytes = chunk_bytes;
  switch (dtype) {
    case pto::kBF16: return pto::loss_ws_bytes<pto::bf16>(c);
    case pto::kF32: return pto::loss_ws_bytes<float>(c);
    default: return 0;
  }
}

int pto_linear_cross_entropy(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const int64_t* targets,
                             int dtype, int64_t rows, int64_t d, int64_t vocab, int64_t ignore_index,
                             double label_smoothing, double z_loss, int reduction, const float* grad_rows, float* loss,
                             float* lse, float* z, void* dhidden, void* dweight, int64_t chunk_bytes, void* workspace,
                             size_t ws_bytes, void* stream) {
  const pto::Call c{hidden, ldh,  weight,         ldw,    targets,   ignore_index, nullptr, nullptr, rows,    d,
                    vocab,  1,    1.0,            label_smoothing,   z_loss,       reduction, grad_rows, loss, lse,
                    z,      dhidden, dweight,     chunk_bytes, "linear_cross_entropy"};
  return pto::run(c, dtype, workspace, ws_bytes, stream);
}

int pto_linear_distillation(const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                            const float* teacher_logits, const int64_t* teacher_index, int dtype, int64_t rows,
                            int64_t d, int64_t vocab, int64_t k, double temperature, int reduction,
                            const float* grad_rows, float* loss, float* lse, float* z, void* dhidden, void* dweight,
                            int64_t chunk_bytes, void* workspace, size_t ws_bytes, void* stream) {
  const pto::Call c{hidden, ldh, weight, ldw, nullptr, 0,   teacher_logits, teacher_index, rows, d,
                    vocab,  k,   temperature, 0.0, 0.0, reduction, grad_rows, loss, lse,
                    z,      dhidden, dweight, chunk_bytes, "linear_distillation"};
  return pto::run(c, dtype, workspace, ws_bytes, stream);
}

int pto_scale(void* x, int dtype, int64_t n, const float* factor, void* stream) {
  PTO_REQUIRE(dtype == pto::kF32 || dtype == pto::kBF16, "scale: unsupported dtype code (fp32 and bf16)");
  PTO_REQUIRE(n >= 0, "scale: negative extent");
  PTO_REQUIRE(n == 0 || (x && factor), "scale: null operand");
  if (n == 0) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = (unsigned)std::min<int64_t>((n + 2047) / 2048, 8 * pto::device_cus());
  if (dtype == pto::kBF16)
    hipLaunchKernelGGL(pto::scale_kernel<pto::bf16>, dim3(blocks), dim3(256), 0, s, static_cast<pto::bf16*>(x), n,
                       factor);
  else
    hipLaunchKernelGGL(pto::scale_kernel<float>, dim3(blocks), dim3(256), 0, s, static_cast<float*>(x), n, factor);
  PTO_LAUNCHED("scale");
  return 0;
}

}  // extern "C"
