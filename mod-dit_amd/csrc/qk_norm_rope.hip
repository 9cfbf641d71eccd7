// Norm of queries and keys with the rotation of their positions in the same pass, and its
// gradient (gfx950).
//
// Of a row x of n values (a head's D, or all heads' H*D of a token):
//   rms:    x^ = x r,          r = (mean(x^2) + eps)^-1/2
//   layer:  x^ = (x - mu) r,   r = (mean((x - mu)^2) + eps)^-1/2
//   y = R(t) (x^ w + b), R(t) turning each pair (a, c) of a head by its angle:
//   (a cos - c sin, c cos + a sin), for the tokens that the tables cover; the others keep x^ w + b.
// Gradient: g = R(t)^T dy; dw = sum g x^, db = sum g over the rows; with d = g w,
//   dx = r (d - x^ mean(d x^) [- mean(d)]).
// x^ is computed again from x rather than kept: x is read for dw anyway.
//
// Bound by HBM: each row is read once and written once. A lane holds 8 elements of a row (one
// 16-byte load, or two of 8 where a pair lies in a head's halves), so D/8 lanes make a row and
// its sums need DPP moves only. All arithmetic is fp32; the result is rounded once.
#include "common.h"

#include <type_traits>

namespace moddit {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxRow = 8192;  // H*D of a norm over all heads

enum { kNone = 0, kRms = 1, kLayer = 2 };

struct RopeTensor {
  const uint16_t* x;
  const uint16_t* dy;
  uint16_t* y;  // y, or dx
  int64_t x_sb, x_sh, x_ss;
  int64_t d_sb, d_sh, d_ss;
  int64_t y_sb, y_sh, y_ss;
  const void* w;
  const void* b;
  int len;
};

struct RopeParams {
  RopeTensor t[2];
  int batch;
  int heads;
  int dim;
  int w_type;  // moddit_dtype of w and b
  int has_bias;  // a bias is added, or its gradient asked for
  float eps;
  const float* cos;
  const float* sin;
  int64_t tab_sb, tab_ss;
  int tab_full;  // 1: D values a row, 0: D/2
  int rope_off, rope_len;
  int tokens;       // the longer of the two lengths
  int token_major;  // a token's heads lie next to each other
  int head_chunk;   // heads of one wave's item
  int head_chunks;
  int64_t items;
  float* partial;  // [q.w, q.b, k.w, k.b][workgroup][row], or null
};

// Sum over the kLanes lanes of a row (8 or 16, aligned), in each of them.
template <int kLanes>
__device__ __forceinline__ float row_sum(float x) {
  auto add = [](float v, auto ctrl) {
    return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x = add(x, std::integral_constant<int, 0xb1>{});   // quad_perm [1,0,3,2]
  x = add(x, std::integral_constant<int, 0x4e>{});   // quad_perm [2,3,0,1]
  x = add(x, std::integral_constant<int, 0x141>{});  // row_half_mirror: the other quad of 8
  if (kLanes == 16) x = add(x, std::integral_constant<int, 0x140>{});  // row_mirror: the other 8
  return x;
}

// Element e (0..7) of lane l of a row: interleaved pairs are (0,1), (2,3), ... of 8 consecutive
// elements; pairs of halves are (e, e + 4) of 4 elements in each half.
template <bool kInter>
__device__ __forceinline__ int col_of(int l, int e, int dim) {
  return kInter ? 8 * l + e : (e < 4 ? 4 * l + e : dim / 2 + 4 * l + e - 4);
}

template <bool kInter>
__device__ __forceinline__ u32x4 load_row(const uint16_t* row, int l, int dim) {
  if (kInter) return *reinterpret_cast<const u32x4*>(row + 8 * l);
  const u32x2 a = *reinterpret_cast<const u32x2*>(row + 4 * l);
  const u32x2 b = *reinterpret_cast<const u32x2*>(row + dim / 2 + 4 * l);
  return u32x4{a.x, a.y, b.x, b.y};
}

template <bool kInter>
__device__ __forceinline__ void store_row(uint16_t* row, int l, int dim, u32x4 v) {
  if (kInter) {
    *reinterpret_cast<u32x4*>(row + 8 * l) = v;
  } else {
    *reinterpret_cast<u32x2*>(row + 4 * l) = u32x2{v.x, v.y};
    *reinterpret_cast<u32x2*>(row + dim / 2 + 4 * l) = u32x2{v.z, v.w};
  }
}

// x, unpacked again from here on: else the compiler keeps the fp32 values of one pass over a row for
// the next, twice the registers of the row itself.
__device__ __forceinline__ void repack(u32x4& x) { asm volatile("" : "+v"(x)); }

template <typename E>
__device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = E::to_float(u16_at(v, e));
}

template <typename E>
__device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
  typename E::vec8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<typename E::elem>(f[i]);  // to nearest even
  return __builtin_bit_cast(u32x4, v);
}

__device__ __forceinline__ float affine_at(const void* w, int type, int64_t i, float none) {
  if (w == nullptr) return none;
  if (type == MODDIT_FP32) return static_cast<const float*>(w)[i];
  const uint16_t u = static_cast<const uint16_t*>(w)[i];
  return type == MODDIT_BF16 ? Bf16::to_float(u) : Fp16::to_float(u);
}

// cos and sin of the lane's four pairs at `token`; 1 and 0 where the tables do not cover it.
// A pair's cos is read at its first element and its sin at its second where a table holds both.
template <bool kInter>
__device__ __forceinline__ void load_angles(const RopeParams& p, int b, int token, int l, float (&c)[4], float (&s)[4]) {
  const int r = token - p.rope_off;
  if (r < 0 || r >= p.rope_len) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
    return;
  }
  const float* cr = p.cos + b * p.tab_sb + r * p.tab_ss;
  const float* sr = p.sin + b * p.tab_sb + r * p.tab_ss;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kInter) {
      c[i] = p.tab_full ? cr[8 * l + 2 * i] : cr[4 * l + i];
      s[i] = p.tab_full ? sr[8 * l + 2 * i + 1] : sr[4 * l + i];
    } else {
      c[i] = cr[4 * l + i];
      s[i] = sr[(p.tab_full ? p.dim / 2 : 0) + 4 * l + i];
    }
  }
}

template <bool kInter, bool kBack>
__device__ __forceinline__ void turn(float (&x)[8], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float& a = x[kInter ? 2 * i : i];
    float& b = x[kInter ? 2 * i + 1 : i + 4];
    const float sn = kBack ? -s[i] : s[i];
    const float a1 = a * c[i] - b * sn;
    b = b * c[i] + a * sn;
    a = a1;
  }
}

// ---- norm over a head's D (or none) ----
// A wave's item is 64 / (D/8) rows at a time: heads of one token where those lie next to each
// other, else tokens of one head; it walks its heads, kUnroll at a time with the loads of q and
// k in flight together, so that a token's angles are read once. 115,200 tokens x 24 heads, D = 128,
// RMS, bf16: 534 us, 5.4 TB/s; gradient of 17,776 x 48, D = 64, layer norm, fp16: 155 us, 4.2 TB/s.
template <int D, typename E, int kNorm, bool kInter, bool kBwd>
__global__ __launch_bounds__(kThreads) void norm_rope_heads_kernel(RopeParams p) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = 64 / kLanes;
  constexpr int kUnroll = kBwd ? 2 : 4;
  constexpr bool kReadX = !kBwd || kNorm != kNone;
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  const int row = lane / kLanes;
  const int l = lane % kLanes;

  float w[2][8], bias[2][8];
  float aw[2][8] = {}, ab[2][8] = {};
  if (kNorm != kNone) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[t][e] = affine_at(p.t[t].w, p.w_type, col_of<kInter>(l, e, D), 1.f);
        bias[t][e] = kBwd ? 0.f : affine_at(p.t[t].b, p.w_type, col_of<kInter>(l, e, D), 0.f);
      }
  }

  const int token_groups = p.token_major ? p.tokens : (p.tokens + kRows - 1) / kRows;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + wave; item < p.items;
       item += static_cast<int64_t>(gridDim.x) * kWaves) {
    const int tg = static_cast<int>(item % token_groups);
    const int rest = static_cast<int>(item / token_groups);
    const int hc = rest % p.head_chunks;
    const int b = rest / p.head_chunks;
    const int token = p.token_major ? tg : tg * kRows + row;
    const int step = p.token_major ? kRows : 1;
    const int h_end = min((hc + 1) * p.head_chunk, p.heads);
    const int h_first = hc * p.head_chunk + (p.token_major ? row : 0);
    float c[4], s[4];
    load_angles<kInter>(p, b, token, l, c, s);
    for (int h0 = h_first; h0 < h_end; h0 += kUnroll * step) {
      u32x4 xr[kUnroll][2], dr[kUnroll][2];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int h = h0 + u * step;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const RopeTensor& q = p.t[t];
          xr[u][t] = dr[u][t] = u32x4{0, 0, 0, 0};
          if (h < h_end && token < q.len) {
            if (kReadX) xr[u][t] = load_row<kInter>(q.x + b * q.x_sb + h * q.x_sh + token * q.x_ss, l, D);
            if (kBwd) dr[u][t] = load_row<kInter>(q.dy + b * q.d_sb + h * q.d_sh + token * q.d_ss, l, D);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int h = h0 + u * step;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const RopeTensor& q = p.t[t];
          float x[8], r = 1.f;
          unpack<E>(xr[u][t], x);
          if (kNorm == kLayer) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += x[e];
            const float mu = row_sum<kLanes>(sum) * (1.f / D);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] -= mu;
          }
          if (kNorm != kNone) {
            float sq = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sq += x[e] * x[e];
            // a row that is not there adds nothing to dw, whatever eps is
            r = h < h_end && token < q.len ? rsqrtf(row_sum<kLanes>(sq) * (1.f / D) + p.eps) : 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= r;
          }
          if (!kBwd) {
            if (kNorm != kNone)
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = x[e] * w[t][e] + bias[t][e];
            turn<kInter, false>(x, c, s);
          } else {
            float g[8];
            unpack<E>(dr[u][t], g);
            turn<kInter, true>(g, c, s);
            if (kNorm == kNone) {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = g[e];
            } else {
              float m1 = 0.f, m2 = 0.f;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                aw[t][e] += g[e] * x[e];
                ab[t][e] += g[e];
                g[e] *= w[t][e];
                m1 += g[e];
                m2 += g[e] * x[e];
              }
              m1 = kNorm == kLayer ? row_sum<kLanes>(m1) * (1.f / D) : 0.f;
              m2 = row_sum<kLanes>(m2) * (1.f / D);
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = r * (g[e] - x[e] * m2 - m1);
            }
          }
          if (h < h_end && token < q.len)
            store_row<kInter>(q.y + b * q.y_sb + h * q.y_sh + token * q.y_ss, l, D, pack<E>(x));
        }
      }
    }
  }

  if constexpr (kBwd && kNorm != kNone) {
    if (p.partial == nullptr) return;
    // the workgroup's sums, one after the other: rows of a wave by shuffles, waves through LDS
    __shared__ float red[kWaves][D];
#pragma unroll
    for (int slot = 0; slot < 4; ++slot) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = slot & 1 ? ab[slot >> 1][e] : aw[slot >> 1][e];
#pragma unroll
        for (int m = kLanes; m < 64; m *= 2) v += __shfl_xor(v, m);
        if (row == 0) red[wave][col_of<kInter>(l, e, D)] = v;
      }
      __syncthreads();
      if (threadIdx.x < D) {
        float v = 0.f;
        for (int i = 0; i < kWaves; ++i) v += red[i][threadIdx.x];
        p.partial[(static_cast<int64_t>(slot) * gridDim.x + blockIdx.x) * D + threadIdx.x] = v;
      }
      __syncthreads();
    }
  }
}

// ---- norm over all heads of a token, forward ----
// One wave per token and tensor at a time, all its loads (kChunks of 16 bytes a lane) in flight
// together and no barrier; the weights wait in LDS as fp32, in two halves of 16 bytes a group of
// 8 elements so that a wave's reads are contiguous. 69,120 tokens x 40 heads, D = 128: 565 us, 5.1 TB/s
// (a workgroup per token, whose sums wait at a barrier: 1,390).
template <int kChunks, typename E, int kNorm, bool kInter, bool kBias>
__global__ __launch_bounds__(kThreads) void norm_rope_wave_kernel(RopeParams p) {
  extern __shared__ float affine[];  // [w, bias][2][n_chunks][4]
  const RopeTensor q = p.t[blockIdx.y];
  const int lanes = p.dim / 8;
  const int n_chunks = p.heads * lanes;
  const float inv_n = 1.f / (p.heads * p.dim);
  for (int i = threadIdx.x; i < n_chunks * 8; i += kThreads) {
    const int ch = i >> 3, e = i & 7;
    const int src = ch / lanes * p.dim + col_of<kInter>(ch % lanes, e, p.dim);
    const int dst = ((e >> 2) * n_chunks + ch) * 4 + (e & 3);
    affine[dst] = affine_at(q.w, p.w_type, src, 1.f);
    if (kBias) affine[8 * n_chunks + dst] = affine_at(q.b, p.w_type, src, 0.f);
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int l = lane % lanes;
  const int h0 = lane / lanes, h_step = 64 / lanes;
  auto wave_sum = [](float x) {
    x = row_sum<16>(x);
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
  };

  const int64_t items = static_cast<int64_t>(p.batch) * q.len;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWaves;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6); item < items; item += step) {
    const int b = static_cast<int>(item / q.len);
    const int token = static_cast<int>(item % q.len);
    const uint16_t* src = q.x + b * q.x_sb + token * q.x_ss + h0 * q.x_sh;
    uint16_t* dst = q.y + b * q.y_sb + token * q.y_ss + h0 * q.y_sh;
    u32x4 raw[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
      raw[j] = lane + 64 * j < n_chunks ? load_row<kInter>(src + j * h_step * q.x_sh, l, p.dim) : u32x4{0, 0, 0, 0};
    float c[4], s[4];
    load_angles<kInter>(p, b, token, l, c, s);
    float mu = 0.f, sq = 0.f;
    if (kNorm == kLayer) {
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        float x[8];
        unpack<E>(raw[j], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) mu += x[e];
      }
      mu = wave_sum(mu) * inv_n;
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      if (kNorm == kLayer) repack(raw[j]);
      float x[8], part = 0.f;
      unpack<E>(raw[j], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) part += (x[e] - mu) * (x[e] - mu);
      if (kNorm != kLayer || lane + 64 * j < n_chunks) sq += part;
    }
    const float r = rsqrtf(wave_sum(sq) * inv_n + p.eps);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int ch = lane + 64 * j;
      if (ch >= n_chunks) break;
      repack(raw[j]);
      float y[8];
      unpack<E>(raw[j], y);
      const f32x4 w[2] = {*reinterpret_cast<const f32x4*>(affine + 4 * ch),
                          *reinterpret_cast<const f32x4*>(affine + 4 * (n_chunks + ch))};
      f32x4 bias[2];
      if (kBias) {
        bias[0] = *reinterpret_cast<const f32x4*>(affine + 4 * (2 * n_chunks + ch));
        bias[1] = *reinterpret_cast<const f32x4*>(affine + 4 * (3 * n_chunks + ch));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = (y[e] - mu) * r * w[e >> 2][e & 3];
        if (kBias) y[e] += bias[e >> 2][e & 3];
      }
      turn<kInter, false>(y, c, s);
      store_row<kInter>(dst + j * h_step * q.y_sh, l, p.dim, pack<E>(y));
    }
  }
}

// ---- norm over all heads of a token, backward ----
// One workgroup per token and tensor at a time; a thread holds kChunks groups of 8 elements, all at
// the same place of their heads (the workgroup's size is a multiple of a row's lanes), and their
// weights across tokens. The next token's rows are loaded before the sums of the current one,
// which wait at a barrier. 28,800 tokens x 40 heads, D = 128: 440 us, 4.0 TB/s, two workgroups a CU by
// registers; a wave per token spills (742 us and more).
template <int kChunks, typename E, int kNorm, bool kInter, bool kBias>
__global__ __launch_bounds__(kThreads) void norm_rope_token_bwd_kernel(RopeParams p) {
  const int which = blockIdx.y;
  const RopeTensor q = p.t[which];
  const int lanes = p.dim / 8;
  const int n_chunks = p.heads * lanes;
  const float inv_n = 1.f / (p.heads * p.dim);
  const int wave = threadIdx.x >> 6;
  const int n_waves = blockDim.x >> 6;
  const int l = threadIdx.x % lanes;
  const int h0 = threadIdx.x / lanes, h_step = blockDim.x / lanes;

  bool ok[kChunks];
  float w[kChunks][8];
  float aw[kChunks][8] = {}, ab[kChunks][8] = {};
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    ok[j] = static_cast<int>(threadIdx.x + j * blockDim.x) < n_chunks;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[j][e] = ok[j] ? affine_at(q.w, p.w_type, (h0 + j * h_step) * p.dim + col_of<kInter>(l, e, p.dim), 1.f) : 0.f;
  }

  __shared__ float red[2][3][kWaves];
  int turn_no = 0;
  // sums over the workgroup; the buffer alternates, so one barrier per call is enough
  auto block_sum = [&](float (&v)[3], int n) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (i >= n) break;
      float x = row_sum<16>(v[i]);
      x += __shfl_xor(x, 16);
      x += __shfl_xor(x, 32);
      if ((threadIdx.x & 63) == 0) red[turn_no][i][wave] = x;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (i >= n) break;
      v[i] = 0.f;
      for (int k = 0; k < n_waves; ++k) v[i] += red[turn_no][i][k];
    }
    turn_no ^= 1;
  };

  const int64_t items = static_cast<int64_t>(p.batch) * q.len;
  u32x4 xn[kChunks], gn[kChunks];
  float cn[4], sn[4];
  auto load = [&](int64_t item) {
    const int b = static_cast<int>(item / q.len);
    const int token = static_cast<int>(item % q.len);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      xn[j] = gn[j] = u32x4{0, 0, 0, 0};
      const int h = h0 + j * h_step;
      if (ok[j]) {
        xn[j] = load_row<kInter>(q.x + b * q.x_sb + h * q.x_sh + token * q.x_ss, l, p.dim);
        gn[j] = load_row<kInter>(q.dy + b * q.d_sb + h * q.d_sh + token * q.d_ss, l, p.dim);
      }
    }
    load_angles<kInter>(p, b, token, l, cn, sn);
  };
  if (blockIdx.x < items) load(blockIdx.x);
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int b = static_cast<int>(item / q.len);
    const int token = static_cast<int>(item % q.len);
    float x[kChunks][8], g[kChunks][8], c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = cn[i];
      s[i] = sn[i];
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      unpack<E>(xn[j], x[j]);
      unpack<E>(gn[j], g[j]);
    }
    if (item + gridDim.x < items) load(item + gridDim.x);
    if (kNorm == kLayer) {
      float v[3] = {};
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[0] += x[j][e];
      block_sum(v, 1);
      const float mu = v[0] * inv_n;
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] = ok[j] ? x[j][e] - mu : 0.f;
    }
    float v[3] = {};
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      turn<kInter, true>(g[j], c, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = g[j][e] * w[j][e];
        v[0] += x[j][e] * x[j][e];
        v[1] += d * x[j][e];
        v[2] += d;
      }
    }
    block_sum(v, kNorm == kLayer ? 3 : 2);
    const float r = rsqrtf(v[0] * inv_n + p.eps);
    const float m2 = v[1] * inv_n * r;                      // mean(d x^)
    const float m1 = kNorm == kLayer ? v[2] * inv_n : 0.f;  // mean(d)
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      if (!ok[j]) continue;
      const int h = h0 + j * h_step;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n = x[j][e] * r;
        aw[j][e] += g[j][e] * n;
        if (kBias) ab[j][e] += g[j][e];
        y[e] = r * (g[j][e] * w[j][e] - n * m2 - m1);
      }
      store_row<kInter>(q.y + b * q.y_sb + h * q.y_sh + token * q.y_ss, l, p.dim, pack<E>(y));
    }
  }

  if (p.partial == nullptr) return;
  const int64_t n = static_cast<int64_t>(p.heads) * p.dim;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    if (!ok[j]) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t i = (h0 + j * h_step) * p.dim + col_of<kInter>(l, e, p.dim);
      p.partial[((which * 2) * static_cast<int64_t>(gridDim.x) + blockIdx.x) * n + i] = aw[j][e];
      if (kBias) p.partial[((which * 2 + 1) * static_cast<int64_t>(gridDim.x) + blockIdx.x) * n + i] = ab[j][e];
    }
  }
}

// Sums over the workgroups' records, in 64 bits and in a fixed order: 64 columns per workgroup,
// the records dealt to its waves: 768 records of 5,120 values, q and k, in 8 us.
struct SumParams {
  const float* partial;
  float* out[4];
  int records;
  int n;
};

__global__ __launch_bounds__(1024) void norm_rope_sum_kernel(SumParams p) {
  __shared__ double red[16][64];
  const int slot = blockIdx.y;
  if (p.out[slot] == nullptr) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = blockIdx.x * 64 + lane;
  double v = 0.0;
  if (col < p.n) {
    const float* at = p.partial + static_cast<int64_t>(slot) * p.records * p.n + col;
    int r = wave;
    for (; r + 7 * 16 < p.records; r += 8 * 16) {  // eight loads in flight
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = at[static_cast<int64_t>(r + 16 * i) * p.n];
#pragma unroll
      for (int i = 0; i < 8; ++i) v += x[i];
    }
    for (; r < p.records; r += 16) v += at[static_cast<int64_t>(r) * p.n];
  }
  red[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && col < p.n) {
    for (int i = 1; i < 16; ++i) v += red[i][lane];
    p.out[slot][col] = static_cast<float>(v);
  }
}

// ---- host side ----
// Workgroups of a backward call, each of which leaves a record of partial sums: enough to fill
// the card, few enough that the records stay small beside the tensors (over all heads 1,536 records
// instead of 768: 527 us in place of 503, 28,800 tokens x 40 heads).
int backward_groups(int64_t work_groups, int across) {
  const int64_t most = across ? 768 : 1536;
  return static_cast<int>(work_groups < 1 ? 1 : (work_groups < most ? work_groups : most));
}

// The waves' items of a call over rows of one head.
void plan_heads(RopeParams& p, int dim) {
  const int rows = 64 / (dim / 8);
  const int64_t groups = static_cast<int64_t>(p.batch) * (p.token_major ? p.tokens : (p.tokens + rows - 1) / rows);
  // all heads in one item unless that leaves the card without work
  int chunk = p.heads;
  const int least = p.token_major ? rows : 1;
  while (chunk > least && groups * ((p.heads + chunk - 1) / chunk) < 4096) chunk = (chunk + 1) / 2;
  if (p.token_major) chunk = (chunk + rows - 1) / rows * rows;
  p.head_chunk = chunk;
  p.head_chunks = (p.heads + chunk - 1) / chunk;
  p.items = groups * p.head_chunks;
}

int64_t groups_of(const RopeParams& p, int across) {
  if (across) return static_cast<int64_t>(p.batch) * p.tokens;
  return (p.items + kWaves - 1) / kWaves;
}

template <typename E, int kNorm, bool kInter, bool kBias>
void launch_wave(const RopeParams& p, int groups, hipStream_t st) {
  const int chunks = p.heads * (p.dim / 8);
  const int per = (chunks + 63) / 64;
  const dim3 grid(groups, 2), block(kThreads);
  const unsigned lds = static_cast<unsigned>(chunks) * 32u * (kBias ? 2u : 1u);  // at most 64 KB
  if (per <= 3)
    hipLaunchKernelGGL((norm_rope_wave_kernel<3, E, kNorm, kInter, kBias>), grid, block, lds, st, p);
  else if (per <= 6)
    hipLaunchKernelGGL((norm_rope_wave_kernel<6, E, kNorm, kInter, kBias>), grid, block, lds, st, p);
  else if (per <= 10)
    hipLaunchKernelGGL((norm_rope_wave_kernel<10, E, kNorm, kInter, kBias>), grid, block, lds, st, p);
  else
    hipLaunchKernelGGL((norm_rope_wave_kernel<16, E, kNorm, kInter, kBias>), grid, block, lds, st, p);
}

template <typename E, int kNorm, bool kInter, bool kBias>
void launch_token_bwd(const RopeParams& p, int groups, hipStream_t st) {
  const int chunks = p.heads * (p.dim / 8);
  const int per = (chunks + kThreads - 1) / kThreads;
  const int threads = ((chunks + per - 1) / per + 63) / 64 * 64;
  const dim3 grid(groups, 2), block(threads);
  if (per == 1)
    hipLaunchKernelGGL((norm_rope_token_bwd_kernel<1, E, kNorm, kInter, kBias>), grid, block, 0, st, p);
  else if (per == 2)
    hipLaunchKernelGGL((norm_rope_token_bwd_kernel<2, E, kNorm, kInter, kBias>), grid, block, 0, st, p);
  else if (per == 3)
    hipLaunchKernelGGL((norm_rope_token_bwd_kernel<3, E, kNorm, kInter, kBias>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((norm_rope_token_bwd_kernel<4, E, kNorm, kInter, kBias>), grid, block, 0, st, p);
}

template <typename E, int kNorm, bool kInter, bool kBwd>
void launch_across(const RopeParams& p, int groups, hipStream_t st) {
  if constexpr (kBwd)
    p.has_bias ? launch_token_bwd<E, kNorm, kInter, true>(p, groups, st) : launch_token_bwd<E, kNorm, kInter, false>(p, groups, st);
  else
    p.has_bias ? launch_wave<E, kNorm, kInter, true>(p, groups, st) : launch_wave<E, kNorm, kInter, false>(p, groups, st);
}

template <typename E, int kNorm, bool kInter, bool kBwd>
void launch_heads(const RopeParams& p, int groups, hipStream_t st) {
  if (p.dim == 128)
    hipLaunchKernelGGL((norm_rope_heads_kernel<128, E, kNorm, kInter, kBwd>), dim3(groups), dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((norm_rope_heads_kernel<64, E, kNorm, kInter, kBwd>), dim3(groups), dim3(kThreads), 0, st, p);
}

template <typename E, bool kInter, bool kBwd>
void launch_norm(const RopeParams& p, int norm, int across, int groups, hipStream_t st) {
  if (across && norm == kRms) return launch_across<E, kRms, kInter, kBwd>(p, groups, st);
  if (across && norm == kLayer) return launch_across<E, kLayer, kInter, kBwd>(p, groups, st);
  if (norm == kRms) return launch_heads<E, kRms, kInter, kBwd>(p, groups, st);
  if (norm == kLayer) return launch_heads<E, kLayer, kInter, kBwd>(p, groups, st);
  launch_heads<E, kNone, kInter, kBwd>(p, groups, st);
}

template <bool kBwd>
void launch_rope(const RopeParams& p, int dtype, int norm, int across, int inter, int groups, hipStream_t st) {
  if (dtype == MODDIT_BF16)
    inter ? launch_norm<Bf16, true, kBwd>(p, norm, across, groups, st) : launch_norm<Bf16, false, kBwd>(p, norm, across, groups, st);
  else
    inter ? launch_norm<Fp16, true, kBwd>(p, norm, across, groups, st) : launch_norm<Fp16, false, kBwd>(p, norm, across, groups, st);
}

bool strides_ok(const int64_t* s) {
  if (s == nullptr) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] % 8) return false;
  return true;
}

// What both directions check, and their parameters but for the tensors' pointers.
int rope_setup(const char* what, RopeParams& p, int batch, int heads, int q_len, int k_len, int head_dim,
               int dtype, int norm, int across, float eps, const void* qw, const void* kw, const void* qb,
               const void* kb, int w_type, const float* cos, const float* sin, const int64_t* tab_strides,
               int tab_dim, int rope_off, int rope_len) {
  MODDIT_CHECK_ARG(batch >= 0 && heads >= 0 && q_len >= 0 && k_len >= 0, "%s: negative size", what);
  if (head_dim != 64 && head_dim != 128) {
    set_error("%s: head_dim must be 64 or 128, got %d", what, head_dim);
    return MODDIT_EUNSUPPORTED;
  }
  if (dtype != MODDIT_BF16 && dtype != MODDIT_FP16) {
    set_error("%s: dtype must be bf16 or fp16", what);
    return MODDIT_EUNSUPPORTED;
  }
  MODDIT_CHECK_ARG(norm >= kNone && norm <= kLayer, "%s: norm must be 0 (none), 1 (rms) or 2 (layer), got %d", what, norm);
  MODDIT_CHECK_ARG(norm != kNone || !(qw || kw || qb || kb || across), "%s: weights, biases and across_heads need a norm", what);
  MODDIT_CHECK_ARG(norm == kNone || (eps >= 0.f && std::isfinite(eps)), "%s: eps must be finite and not negative", what);
  MODDIT_CHECK_ARG(w_type >= MODDIT_BF16 && w_type <= MODDIT_FP32, "%s: weight dtype must be bf16, fp16 or fp32", what);
  if (across && static_cast<int64_t>(heads) * head_dim > kMaxRow) {
    set_error("%s: a norm over all heads takes heads * head_dim <= %d, got %lld", what, kMaxRow,
              static_cast<long long>(heads) * head_dim);
    return MODDIT_EUNSUPPORTED;
  }
  MODDIT_CHECK_ARG(rope_off >= 0 && rope_len >= 0, "%s: rope offset and length must not be negative", what);
  if (rope_len > 0) {
    MODDIT_CHECK_ARG(cos && sin && tab_strides, "%s: rotation tables missing", what);
    MODDIT_CHECK_ARG(tab_dim == head_dim || tab_dim == head_dim / 2, "%s: tables must hold head_dim or head_dim / 2 values a row, got %d", what, tab_dim);
    MODDIT_CHECK_ARG(tab_strides[0] >= 0 && tab_strides[1] >= 0, "%s: table strides must not be negative", what);
    MODDIT_CHECK_ARG(static_cast<int64_t>(rope_off) + rope_len <= (q_len < k_len ? q_len : k_len),
                     "%s: rotated tokens [%d, %lld) exceed the %d tokens of the shorter tensor", what, rope_off,
                     static_cast<long long>(rope_off) + rope_len, q_len < k_len ? q_len : k_len);
  }
  p.batch = batch;
  p.heads = heads;
  p.dim = head_dim;
  p.w_type = w_type;
  p.eps = eps;
  p.cos = cos;
  p.sin = sin;
  p.tab_sb = rope_len > 0 ? tab_strides[0] : 0;
  p.tab_ss = rope_len > 0 ? tab_strides[1] : 0;
  p.tab_full = tab_dim == head_dim;
  p.rope_off = rope_off;
  p.rope_len = rope_len;
  p.tokens = q_len > k_len ? q_len : k_len;
  p.t[0].w = qw;
  p.t[1].w = kw;
  p.has_bias = qb != nullptr || kb != nullptr;
  p.t[0].b = qb;
  p.t[1].b = kb;
  p.t[0].len = q_len;
  p.t[1].len = k_len;
  p.partial = nullptr;
  return MODDIT_OK;
}

void set_strides(int64_t& b, int64_t& h, int64_t& s, const int64_t* v) {
  b = v[0];
  h = v[1];
  s = v[2];
}

}  // namespace
}  // namespace moddit

extern "C" int moddit_qk_norm_rope(const void* q, const void* k, void* q_out, void* k_out, int batch, int heads,
                                   int q_len, int k_len, int head_dim, const int64_t q_strides[3],
                                   const int64_t k_strides[3], const int64_t qo_strides[3],
                                   const int64_t ko_strides[3], int dtype, int norm, int across_heads, float eps,
                                   const void* q_weight, const void* k_weight, const void* q_bias,
                                   const void* k_bias, int weight_dtype, const float* cos, const float* sin,
                                   const int64_t table_strides[2], int table_dim, int rope_offset, int rope_len,
                                   int interleaved, moddit_stream_t stream) {
  using namespace moddit;
  clear_error();
  RopeParams p;
  if (const int rc = rope_setup("qk_norm_rope", p, batch, heads, q_len, k_len, head_dim, dtype, norm, across_heads,
                                eps, q_weight, k_weight, q_bias, k_bias, weight_dtype, cos, sin, table_strides,
                                table_dim, rope_offset, rope_len))
    return rc;
  MODDIT_CHECK_ARG(strides_ok(q_strides) && strides_ok(k_strides) && strides_ok(qo_strides) && strides_ok(ko_strides),
                   "qk_norm_rope: strides must be non-negative multiples of 8 elements");
  if (batch == 0 || heads == 0 || p.tokens == 0) return MODDIT_OK;
  MODDIT_CHECK_ARG((q_len == 0 || (q && q_out)) && (k_len == 0 || (k && k_out)), "qk_norm_rope: null tensor pointer");
  MODDIT_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(q_out) && aligned16(k_out),
                   "qk_norm_rope: tensors must be 16-byte aligned");
  const void* x[2] = {q, k};
  void* y[2] = {q_out, k_out};
  const int64_t* xs[2] = {q_strides, k_strides};
  const int64_t* ys[2] = {qo_strides, ko_strides};
  for (int t = 0; t < 2; ++t) {
    p.t[t].x = static_cast<const uint16_t*>(x[t]);
    p.t[t].dy = nullptr;
    p.t[t].y = static_cast<uint16_t*>(y[t]);
    set_strides(p.t[t].x_sb, p.t[t].x_sh, p.t[t].x_ss, xs[t]);
    set_strides(p.t[t].d_sb, p.t[t].d_sh, p.t[t].d_ss, xs[t]);
    set_strides(p.t[t].y_sb, p.t[t].y_sh, p.t[t].y_ss, ys[t]);
  }
  p.token_major = q_strides[1] < q_strides[2];
  plan_heads(p, head_dim);
  int64_t groups = groups_of(p, across_heads);
  if (across_heads) {  // a wave walks several tokens, so that the weights are read to LDS seldom
    groups = (groups + kWaves - 1) / kWaves;
    if (groups > 1280) groups = 1280;
  }
  MODDIT_CHECK_ARG(groups <= 0x7fffffff, "qk_norm_rope: too many tokens");
  launch_rope<false>(p, dtype, norm, across_heads, interleaved, static_cast<int>(groups), as_stream(stream));
  MODDIT_CHECK_LAUNCH("qk_norm_rope");
  return MODDIT_OK;
}

extern "C" int64_t moddit_qk_norm_rope_bwd_workspace_floats(int batch, int heads, int q_len, int k_len, int head_dim,
                                                            int across_heads) {
  using namespace moddit;
  if (batch <= 0 || heads <= 0 || q_len < 0 || k_len < 0 || (head_dim != 64 && head_dim != 128)) return 0;
  // an upper bound whatever the strides: as many records as a call may leave
  const int64_t tokens = static_cast<int64_t>(batch) * (q_len > k_len ? q_len : k_len);
  const int64_t records = backward_groups(across_heads ? tokens : tokens * heads, across_heads);
  return 4 * records * (across_heads ? static_cast<int64_t>(heads) * head_dim : head_dim);
}

extern "C" int moddit_qk_norm_rope_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, void* dq,
                                       void* dk, float* dq_weight, float* dk_weight, float* dq_bias, float* dk_bias,
                                       int batch, int heads, int q_len, int k_len, int head_dim,
                                       const int64_t q_strides[3], const int64_t k_strides[3],
                                       const int64_t dqo_strides[3], const int64_t dko_strides[3],
                                       const int64_t dq_strides[3], const int64_t dk_strides[3], int dtype, int norm,
                                       int across_heads, float eps, const void* q_weight, const void* k_weight,
                                       int weight_dtype, const float* cos, const float* sin,
                                       const int64_t table_strides[2], int table_dim, int rope_offset, int rope_len,
                                       int interleaved, float* workspace, int64_t workspace_floats,
                                       moddit_stream_t stream) {
  using namespace moddit;
  clear_error();
  RopeParams p;
  if (const int rc = rope_setup("qk_norm_rope_bwd", p, batch, heads, q_len, k_len, head_dim, dtype, norm, across_heads,
                                eps, q_weight, k_weight, nullptr, nullptr, weight_dtype, cos, sin, table_strides,
                                table_dim, rope_offset, rope_len))
    return rc;
  MODDIT_CHECK_ARG(strides_ok(q_strides) && strides_ok(k_strides) && strides_ok(dqo_strides) &&
                       strides_ok(dko_strides) && strides_ok(dq_strides) && strides_ok(dk_strides),
                   "qk_norm_rope_bwd: strides must be non-negative multiples of 8 elements");
  const bool sums = dq_weight || dk_weight || dq_bias || dk_bias;
  MODDIT_CHECK_ARG(!sums || norm != kNone, "qk_norm_rope_bwd: gradients of weights and biases need a norm");
  if (batch == 0 || heads == 0 || p.tokens == 0) return MODDIT_OK;
  MODDIT_CHECK_ARG((q_len == 0 || (dq_out && dq && (q || norm == kNone))) &&
                       (k_len == 0 || (dk_out && dk && (k || norm == kNone))),
                   "qk_norm_rope_bwd: null tensor pointer");
  MODDIT_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(dq_out) && aligned16(dk_out) && aligned16(dq) && aligned16(dk),
                   "qk_norm_rope_bwd: tensors must be 16-byte aligned");
  const void* x[2] = {q, k};
  const void* d[2] = {dq_out, dk_out};
  void* y[2] = {dq, dk};
  const int64_t* xs[2] = {q_strides, k_strides};
  const int64_t* ds[2] = {dqo_strides, dko_strides};
  const int64_t* ys[2] = {dq_strides, dk_strides};
  for (int t = 0; t < 2; ++t) {
    p.t[t].x = static_cast<const uint16_t*>(x[t]);
    p.t[t].dy = static_cast<const uint16_t*>(d[t]);
    p.t[t].y = static_cast<uint16_t*>(y[t]);
    set_strides(p.t[t].x_sb, p.t[t].x_sh, p.t[t].x_ss, xs[t]);
    set_strides(p.t[t].d_sb, p.t[t].d_sh, p.t[t].d_ss, ds[t]);
    set_strides(p.t[t].y_sb, p.t[t].y_sh, p.t[t].y_ss, ys[t]);
  }
  p.token_major = q_strides[1] < q_strides[2];
  plan_heads(p, head_dim);
  const int groups = backward_groups(groups_of(p, across_heads), across_heads);
  const int64_t row = across_heads ? static_cast<int64_t>(heads) * head_dim : head_dim;
  if (sums) {
    MODDIT_CHECK_ARG(workspace != nullptr && workspace_floats >= 4 * groups * row,
                     "qk_norm_rope_bwd: workspace of %lld floats, %lld needed", static_cast<long long>(workspace_floats),
                     static_cast<long long>(4 * groups * row));
    p.partial = workspace;
    p.has_bias = dq_bias != nullptr || dk_bias != nullptr;
  }
  hipStream_t st = as_stream(stream);
  launch_rope<true>(p, dtype, norm, across_heads, interleaved, groups, st);
  MODDIT_CHECK_LAUNCH("qk_norm_rope_bwd");
  if (sums) {
    SumParams sp{workspace, {dq_weight, dq_bias, dk_weight, dk_bias}, groups, static_cast<int>(row)};
    hipLaunchKernelGGL(norm_rope_sum_kernel, dim3(static_cast<unsigned>((row + 63) / 64), 4), dim3(1024), 0, st, sp);
    MODDIT_CHECK_LAUNCH("qk_norm_rope_bwd (sums)");
  }
  return MODDIT_OK;
}
