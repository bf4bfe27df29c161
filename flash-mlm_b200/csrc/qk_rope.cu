// Per-head norm of queries and keys with the position rotation in the same
// pass, forward and backward.
//
//   xh = x * rstd, rstd = 1 / sqrt(mean(x^2) + eps);  y = R(pos) (xh * w)
//   g = R(pos)^T dy;  dw = sum_rows g * xh;  dx = rstd * (g w - xh * mean(g w xh))
//
// Bound by HBM: x is read once and y written once (backward: x and dy read, dx
// written); everything else stays in registers.  A row is held by D / 16
// lanes, 16 columns each in two 16-byte vectors, chosen so that both members
// of every rotated pair are in one lane: of the R / 8 rotated vectors, lane l
// takes l and l + R / 16; the unrotated rest goes to the remaining lanes.  The
// row sums are shuffles over those lanes.  A lane group walks the heads of one
// token, so the token's cosines and sines, which are the same for every head,
// are loaded once.  All arithmetic is in 32 bits; outputs are rounded once.
//
// What keeps memory busy is the loads that each thread has under way: four
// heads at a time forward, two backward, and the registers for them rather than
// more warps.  16 x 4096 tokens, 32 + 8 heads of 128, a projection's strides:
// forward 222 us (6.0 TB/s; with registers capped for two blocks per SM 254,
// two heads at a time 268, eight 282), backward 388 us (5.2 TB/s; weights in
// registers 421, one head at a time and three blocks 445).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace fmlm {
namespace {

constexpr int kErrPosition = 6;
constexpr int kThreads = 256;
constexpr int kBwdBlocksMax = 148 * 4;  // per tensor; also the rows of the partial-sum workspace

struct RopeParams {
  const uint16_t *x[2], *g[2];  // q, k and the gradients of their outputs
  long long xs[2][3], gs[2][3]; // batch, head, row strides in elements
  uint16_t* out[2];
  const void* w[2];
  float* part[2];               // backward: partial weight gradients [blocks][D]
  int heads[2];
  int head_step;                // heads per block
  int splits[2];                // head ranges per tensor
  int packed, normalize, weight_f32, want_dw;
  int B, N, R, max_pos;
  long long tokens;             // B * N, or T packed
  float eps;
  const float* table;
  const int* positions;
  const int* offsets;
  const int* lengths;
  const long long* token_idx;
  int* err;
};

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float2 t;
    if constexpr (BF16) t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[e]));
    else t = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
    f[2 * e] = t.x;
    f[2 * e + 1] = t.y;
  }
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint32_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (BF16) {
      __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
      u[e] = *reinterpret_cast<uint32_t*>(&t);
    } else {
      __half2 t = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
      u[e] = *reinterpret_cast<uint32_t*>(&t);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// The token a lane group works on: where its rows are and how it is rotated.
struct Token {
  long long b, n;  // batch and row coordinates in x (packed: 0, token)
  int pos;
  bool valid;
};

template <int D>
__device__ __forceinline__ Token locate(const RopeParams& p, long long i) {
  Token t;
  int seq, idx;
  if (p.packed) {
    const long long flat = __ldg(p.token_idx + i);
    if (flat >> 31) {
      seq = (int)(flat / p.N);
      idx = (int)(flat % p.N);
    } else {
      seq = (unsigned)flat / (unsigned)p.N;
      idx = (unsigned)flat % (unsigned)p.N;
    }
    seq = min(max(seq, 0), p.B - 1);
    t.b = 0;
    t.n = i;
    t.valid = true;
  } else {
    if (i >> 31) {
      seq = (int)(i / p.N);
      idx = (int)(i % p.N);
    } else {
      seq = (unsigned)i / (unsigned)p.N;
      idx = (unsigned)i % (unsigned)p.N;
    }
    t.b = seq;
    t.n = idx;
    t.valid = p.lengths == nullptr || idx < __ldg(p.lengths + seq);
  }
  t.pos = 0;
  if (t.valid && p.R > 0) {
    // (an index and an offset may pass 32 bits together)
    const long long pos = p.positions ? __ldg(p.positions + i) : (long long)idx + (p.offsets ? __ldg(p.offsets + seq) : 0);
    if (pos < 0 || pos >= p.max_pos) atomicExch(p.err, kErrPosition);
    t.pos = (int)min(max(pos, 0ll), (long long)p.max_pos - 1);
  }
  return t;
}

// Lane l's two vectors of a row, as column offsets.
__device__ __forceinline__ void lane_columns(int R, int l, int& c0, int& c1) {
  const int r = R / 16;
  if (l < r) {
    c0 = l * 8;
    c1 = (l + r) * 8;
  } else {
    c0 = R + (l - r) * 16;
    c1 = c0 + 8;
  }
}

// Cosines and sines of the lane's eight pairs (1 and 0 where nothing turns).
template <bool HALF>
__device__ __forceinline__ void load_turns(const RopeParams& p, int pos, int l, int c0, int c1, float* cs, float* sn) {
  if (l < p.R / 16) {
    const float4* row = reinterpret_cast<const float4*>(p.table + (long long)pos * p.R);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // HALF: pairs c0 .. c0 + 7.  Interleaved: pairs c0 / 2 .. + 3 and c1 / 2 .. + 3.
      const float4 v = __ldg(row + (HALF ? c0 / 2 + e : (e < 2 ? c0 / 4 + e : c1 / 4 + e - 2)));
      cs[2 * e] = v.x;
      sn[2 * e] = v.y;
      cs[2 * e + 1] = v.z;
      sn[2 * e + 1] = v.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = 1.f;
      sn[e] = 0.f;
    }
  }
}

// v[0..7] and v[8..15] are the lane's vectors: turn its eight pairs.
template <bool HALF>
__device__ __forceinline__ void turn(float* v, const float* cs, const float* sn) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = HALF ? e : 2 * e, j = HALF ? e + 8 : 2 * e + 1;
    const float a = v[i], b = v[j];
    v[i] = fmaf(a, cs[e], -(b * sn[e]));
    v[j] = fmaf(b, cs[e], a * sn[e]);
  }
}

template <bool BF16>
__device__ __forceinline__ void load_weights(const RopeParams& p, const void* w, int c0, int c1, float* f) {
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] = 1.f;
  } else if (p.weight_f32) {
    const float* s = reinterpret_cast<const float*>(w);
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] = __ldg(s + (e < 8 ? c0 + e : c1 + e - 8));
  } else {
    const uint16_t* s = reinterpret_cast<const uint16_t*>(w);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint16_t u = __ldg(s + (e < 8 ? c0 + e : c1 + e - 8));
      if constexpr (BF16) f[e] = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(&u));
      else f[e] = __half2float(*reinterpret_cast<const __half*>(&u));
    }
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float s) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <int D, bool HALF, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) qk_rope_fwd_kernel(const RopeParams p) {
  constexpr int LPR = D / 16, UNROLL = 4;
  const int l = threadIdx.x % LPR;
  const long long i = (long long)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int which = (int)blockIdx.y < p.splits[0] ? 0 : 1;
  const int h0 = ((int)blockIdx.y - (which ? p.splits[0] : 0)) * p.head_step;
  const int h1 = min(h0 + p.head_step, p.heads[which]);
  const bool in = i < p.tokens;
  Token t{0, 0, 0, false};
  if (in) t = locate<D>(p, i);
  int c0, c1;
  lane_columns(p.R, l, c0, c1);
  float cs[8], sn[8], w[16];
  load_turns<HALF>(p, t.pos, t.valid ? l : LPR, c0, c1, cs, sn);
  load_weights<BF16>(p, p.w[which], c0, c1, w);
  const uint16_t* x = p.x[which] + t.b * p.xs[which][0] + t.n * p.xs[which][2];
  const long long sh = p.xs[which][1];
  uint16_t* y = p.out[which] + (p.packed ? t.n : t.b * p.heads[which] * p.N + t.n) * D;
  const long long oh = (p.packed ? p.tokens : p.N) * D;
  for (int h = h0; h < h1; h += UNROLL) {
    uint4 a[UNROLL], b[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      a[u] = b[u] = make_uint4(0, 0, 0, 0);
      if (t.valid && h + u < h1) {
        a[u] = __ldg(reinterpret_cast<const uint4*>(x + (h + u) * sh + c0));
        b[u] = __ldg(reinterpret_cast<const uint4*>(x + (h + u) * sh + c1));
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float v[16];
      unpack8<BF16>(a[u], v);
      unpack8<BF16>(b[u], v + 8);
      if (p.normalize) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) s = fmaf(v[e], v[e], s);
        s = row_sum<LPR>(s);
        const float rstd = t.valid ? rsqrtf(s * (1.f / D) + p.eps) : 0.f;  // a padding row stays 0 (eps may be 0)
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= rstd * w[e];
      }
      turn<HALF>(v, cs, sn);
      if (in && h + u < h1) {
        *reinterpret_cast<uint4*>(y + (h + u) * oh + c0) = pack8<BF16>(v);
        *reinterpret_cast<uint4*>(y + (h + u) * oh + c1) = pack8<BF16>(v + 8);
      }
    }
  }
}

// Blocks walk token tiles with a stride of the grid, keeping their share of
// the weights' gradient in registers; each ends with one row of partial sums.
template <int D, bool HALF, bool BF16>
__global__ void __launch_bounds__(kThreads, 2) qk_rope_bwd_kernel(const RopeParams p) {
  constexpr int LPR = D / 16, UNROLL = 2, TOK = kThreads / LPR;
  __shared__ float red[kThreads / 32][D];
  const int l = threadIdx.x % LPR;
  const int which = (int)blockIdx.y < p.splits[0] ? 0 : 1;
  const int split = (int)blockIdx.y - (which ? p.splits[0] : 0);
  const int h0 = split * p.head_step;
  const int h1 = min(h0 + p.head_step, p.heads[which]);
  int c0, c1;
  lane_columns(p.R, l, c0, c1);
  // the lanes' weights in shared memory (rows of 80 bytes: no two lanes of a
  // row on the same bank): 16 registers fewer than holding them
  __shared__ float4 sw[LPR][5];
  if (threadIdx.x < LPR) {
    float w0[16];
    load_weights<BF16>(p, p.w[which], c0, c1, w0);
#pragma unroll
    for (int e = 0; e < 4; ++e) sw[l][e] = make_float4(w0[4 * e], w0[4 * e + 1], w0[4 * e + 2], w0[4 * e + 3]);
  }
  __syncthreads();
  float dw[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[e] = 0.f;
  const long long sh = p.xs[which][1], gh = p.gs[which][1];
  const long long oh = (p.packed ? p.tokens : p.N) * D;
  for (long long base = (long long)blockIdx.x * TOK; base < p.tokens; base += (long long)gridDim.x * TOK) {
    const long long i = base + threadIdx.x / LPR;
    const bool in = i < p.tokens;
    Token t{0, 0, 0, false};
    if (in) t = locate<D>(p, i);
    float cs[8], sn[8];
    load_turns<HALF>(p, t.pos, t.valid ? l : LPR, c0, c1, cs, sn);
#pragma unroll
    for (int e = 0; e < 8; ++e) sn[e] = -sn[e];  // the transposed rotation
    const uint16_t* x = p.x[which] + t.b * p.xs[which][0] + t.n * p.xs[which][2];
    const uint16_t* g = p.g[which] + t.b * p.gs[which][0] + t.n * p.gs[which][2];
    uint16_t* y = p.out[which] + (p.packed ? t.n : t.b * p.heads[which] * p.N + t.n) * D;
    for (int h = h0; h < h1; h += UNROLL) {
      uint4 a[UNROLL], b[UNROLL], ga[UNROLL], gb[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        a[u] = b[u] = ga[u] = gb[u] = make_uint4(0, 0, 0, 0);
        if (t.valid && h + u < h1) {
          if (p.normalize) {
            a[u] = __ldg(reinterpret_cast<const uint4*>(x + (h + u) * sh + c0));
            b[u] = __ldg(reinterpret_cast<const uint4*>(x + (h + u) * sh + c1));
          }
          ga[u] = __ldg(reinterpret_cast<const uint4*>(g + (h + u) * gh + c0));
          gb[u] = __ldg(reinterpret_cast<const uint4*>(g + (h + u) * gh + c1));
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        float v[16], d[16];
        unpack8<BF16>(ga[u], d);
        unpack8<BF16>(gb[u], d + 8);
        turn<HALF>(d, cs, sn);
        if (p.normalize) {
          unpack8<BF16>(a[u], v);
          unpack8<BF16>(b[u], v + 8);
          float w[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 x4 = sw[l][e];
            w[4 * e] = x4.x; w[4 * e + 1] = x4.y; w[4 * e + 2] = x4.z; w[4 * e + 3] = x4.w;
          }
          float s = 0.f, c = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s = fmaf(v[e], v[e], s);
            c = fmaf(d[e] * w[e], v[e], c);
          }
          s = row_sum<LPR>(s);
          c = row_sum<LPR>(c);
          const float rstd = t.valid && h + u < h1 ? rsqrtf(s * (1.f / D) + p.eps) : 0.f;
          c *= rstd * (1.f / D);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float xh = v[e] * rstd;
            dw[e] = fmaf(d[e], xh, dw[e]);
            d[e] = rstd * fmaf(d[e], w[e], -(xh * c));
          }
        }
        if (in && h + u < h1) {
          *reinterpret_cast<uint4*>(y + (h + u) * oh + c0) = pack8<BF16>(d);
          *reinterpret_cast<uint4*>(y + (h + u) * oh + c1) = pack8<BF16>(d + 8);
        }
      }
    }
  }
  if (!p.want_dw) return;
  // lane groups of a warp, then warps, in a fixed order
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) dw[e] += __shfl_xor_sync(0xffffffffu, dw[e], o);
  }
  if ((threadIdx.x & 31) < LPR) {
#pragma unroll
    for (int e = 0; e < 16; ++e) red[threadIdx.x >> 5][e < 8 ? c0 + e : c1 + e - 8] = dw[e];
  }
  __syncthreads();
  float* dst = p.part[which] + ((long long)split * gridDim.x + blockIdx.x) * D;
  for (int c = threadIdx.x; c < D; c += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kThreads / 32; ++k) s += red[k][c];
    dst[c] = s;
  }
}

// Sums the partial rows in a fixed order: one block per tensor and 8 columns,
// 32 threads a column, then a shuffle.
template <bool BF16>
__global__ void __launch_bounds__(256) qk_rope_dw_kernel(const float* part0, const float* part1, int rows0, int rows1,
                                                         int D, void* dw0, void* dw1, int f32) {
  const int which = blockIdx.y;
  const float* part = which ? part1 : part0;
  void* dw = which ? dw1 : dw0;
  if (dw == nullptr) return;
  const int rows = which ? rows1 : rows0;
  const int c = blockIdx.x * 8 + (threadIdx.x & 7), r0 = threadIdx.x >> 3;
  __shared__ float red[32][9];
  float s = 0.f;
  for (int r = r0; r < rows; r += 32) s += part[(long long)r * D + c];
  red[r0][threadIdx.x & 7] = s;
  __syncthreads();
  const int lane = threadIdx.x & 31, col = threadIdx.x >> 5;
  s = red[lane][col];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) {
    const int oc = blockIdx.x * 8 + col;
    if (f32) reinterpret_cast<float*>(dw)[oc] = s;
    else if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(dw)[oc] = __float2bfloat16_rn(s);
    else reinterpret_cast<__half*>(dw)[oc] = __float2half_rn(s);
  }
}

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

template <int D, bool HALF, bool BF16>
int launch(RopeParams p, const fmlm_qk_rope_args* a, bool bwd, cudaStream_t s) {
  constexpr int TOK = kThreads / (D / 16);
  const long long tiles = (p.tokens + TOK - 1) / TOK;
  if (tiles > 0x7fffffffLL) return set_error(FMLM_ERR_INVALID, "problem too large");
  const int maxh = std::max(p.heads[0], p.heads[1]);
  // Heads per block: as many as leave the GPU several blocks per SM, so that a
  // token's cosines and sines serve many heads when there are many tokens and
  // single tokens still spread over the GPU.
  const long long want = (long long)device_sm_count() * 4;
  int step = maxh;
  while (step > 1 && tiles * (ceil_div(p.heads[0], step) + ceil_div(p.heads[1], step)) < want) step = (step + 1) / 2;
  p.head_step = step;
  p.splits[0] = ceil_div(p.heads[0], step);
  p.splits[1] = ceil_div(p.heads[1], step);
  const unsigned ny = (unsigned)(p.splits[0] + p.splits[1]);
  if (ny > 65535) return set_error(FMLM_ERR_INVALID, "too many heads");
  if (!bwd) {
    qk_rope_fwd_kernel<D, HALF, BF16><<<dim3((unsigned)tiles, ny), kThreads, 0, s>>>(p);
    return check_launch("qk_rope_fwd_kernel");
  }
  // Blocks per head range: the partial sums of one tensor fit the workspace.
  const int cap = std::max(1, kBwdBlocksMax / std::max(p.splits[0], p.splits[1]));
  const unsigned nx = (unsigned)std::min<long long>(tiles, cap);
  qk_rope_bwd_kernel<D, HALF, BF16><<<dim3(nx, ny), kThreads, 0, s>>>(p);
  int rc = check_launch("qk_rope_bwd_kernel");
  if (rc || !p.want_dw) return rc;
  qk_rope_dw_kernel<BF16><<<dim3(D / 8, 2), 256, 0, s>>>(p.part[0], p.part[1], p.splits[0] * nx, p.splits[1] * nx, D,
                                                         a->dq_weight, a->dk_weight, a->weight_f32);
  return check_launch("qk_rope_dw_kernel");
}

template <bool HALF, bool BF16>
int dispatch(const RopeParams& p, const fmlm_qk_rope_args* a, bool bwd, cudaStream_t s) {
  switch (a->head_dim) {
    case 16: return launch<16, HALF, BF16>(p, a, bwd, s);
    case 32: return launch<32, HALF, BF16>(p, a, bwd, s);
    case 64: return launch<64, HALF, BF16>(p, a, bwd, s);
    case 128: return launch<128, HALF, BF16>(p, a, bwd, s);
    case 256: return launch<256, HALF, BF16>(p, a, bwd, s);
    default: return set_error(FMLM_ERR_UNSUPPORTED, "HEAD_DIM must be one of {16, 32, 64, 128, 256}");
  }
}

int check_rows(const fmlm_view4& v, const char* name) {
  if (!v.data || !aligned16(v.data)) return set_error(FMLM_ERR_INVALID, "%s must be a 16-byte aligned device pointer", name);
  if (v.batch_stride % 8 || v.head_stride % 8 || v.row_stride % 8)
    return set_error(FMLM_ERR_INVALID, "%s: strides must be multiples of 8 elements", name);
  return FMLM_OK;
}

int run(const fmlm_qk_rope_args* a, bool bwd, void* stream) {
  if (!a) return set_error(FMLM_ERR_INVALID, "null args");
  if (a->dtype != FMLM_DTYPE_F16 && a->dtype != FMLM_DTYPE_BF16) return set_error(FMLM_ERR_INVALID, "dtype must be f16 or bf16");
  if (a->q_heads < 1 || a->k_heads < 1 || a->batch < 1 || a->seq_len < 1)
    return set_error(FMLM_ERR_INVALID, "batch, seq_len, q_heads and k_heads must be >= 1");
  if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 16 != 0)
    return set_error(FMLM_ERR_INVALID, "rotary_dim must be a multiple of 16 in [0, head_dim]");
  if (a->pairs != FMLM_PAIRS_HALF && a->pairs != FMLM_PAIRS_INTERLEAVED) return set_error(FMLM_ERR_INVALID, "bad pairs");
  if (a->rotary_dim > 0 && (!a->table || !aligned16(a->table) || a->max_positions < 1))
    return set_error(FMLM_ERR_INVALID, "a rotation needs a 16-byte aligned table of at least one position");
  if (a->positions && a->position_offsets) return set_error(FMLM_ERR_INVALID, "give positions or position_offsets");
  if (a->packed && !a->token_indices) return set_error(FMLM_ERR_INVALID, "packed rows need token_indices");
  if (!a->normalize && (a->q_weight || a->k_weight || a->dq_weight || a->dk_weight))
    return set_error(FMLM_ERR_INVALID, "weights need normalize");
  if (!a->error_word) return set_error(FMLM_ERR_INVALID, "error_word is required");
  if (!a->q_out || !a->k_out || !aligned16(a->q_out) || !aligned16(a->k_out))
    return set_error(FMLM_ERR_INVALID, "q_out and k_out are required and 16-byte aligned");
  int rc;
  if ((rc = check_rows(a->q, "q")) || (rc = check_rows(a->k, "k"))) return rc;
  if (bwd && ((rc = check_rows(a->gq, "gq")) || (rc = check_rows(a->gk, "gk")))) return rc;
  RopeParams p{};
  const fmlm_view4 *x[2] = {&a->q, &a->k}, *g[2] = {&a->gq, &a->gk};
  for (int i = 0; i < 2; ++i) {
    p.x[i] = reinterpret_cast<const uint16_t*>(x[i]->data);
    p.xs[i][0] = x[i]->batch_stride;
    p.xs[i][1] = x[i]->head_stride;
    p.xs[i][2] = x[i]->row_stride;
    p.g[i] = reinterpret_cast<const uint16_t*>(g[i]->data);
    p.gs[i][0] = g[i]->batch_stride;
    p.gs[i][1] = g[i]->head_stride;
    p.gs[i][2] = g[i]->row_stride;
  }
  p.out[0] = reinterpret_cast<uint16_t*>(a->q_out);
  p.out[1] = reinterpret_cast<uint16_t*>(a->k_out);
  p.w[0] = a->q_weight;
  p.w[1] = a->k_weight;
  p.heads[0] = a->q_heads;
  p.heads[1] = a->k_heads;
  p.packed = a->packed != 0;
  p.normalize = a->normalize != 0;
  p.weight_f32 = a->weight_f32 != 0;
  p.want_dw = bwd && (a->dq_weight || a->dk_weight);
  p.B = a->batch;
  p.N = a->seq_len;
  p.R = a->rotary_dim;
  p.max_pos = a->max_positions;
  p.tokens = a->packed ? a->q.rows : (long long)a->batch * a->seq_len;
  p.eps = a->eps;
  p.table = a->table;
  p.positions = a->positions;
  p.offsets = a->position_offsets;
  p.lengths = a->packed ? nullptr : a->lengths;
  p.token_idx = reinterpret_cast<const long long*>(a->token_indices);
  p.err = a->error_word;
  if (a->packed && (a->q.rows < 1 || a->k.rows != a->q.rows))
    return set_error(FMLM_ERR_INVALID, "packed q and k must have the same number (>= 1) of rows");
  if (p.want_dw) {
    if (!a->workspace || a->workspace_bytes < fmlm_qk_rope_bwd_workspace_bytes(a->head_dim))
      return set_error(FMLM_ERR_INVALID, "workspace too small (%zu bytes needed)",
                       fmlm_qk_rope_bwd_workspace_bytes(a->head_dim));
    p.part[0] = reinterpret_cast<float*>(a->workspace);
    p.part[1] = p.part[0] + (size_t)kBwdBlocksMax * a->head_dim;
    if (std::max(a->q_heads, a->k_heads) > kBwdBlocksMax) return set_error(FMLM_ERR_INVALID, "too many heads");
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool half = a->pairs == FMLM_PAIRS_HALF;
  if (a->dtype == FMLM_DTYPE_BF16) return half ? dispatch<true, true>(p, a, bwd, s) : dispatch<false, true>(p, a, bwd, s);
  return half ? dispatch<true, false>(p, a, bwd, s) : dispatch<false, false>(p, a, bwd, s);
}

}  // namespace
}  // namespace fmlm

extern "C" size_t fmlm_qk_rope_bwd_workspace_bytes(int32_t head_dim) {
  return (size_t)2 * fmlm::kBwdBlocksMax * (head_dim > 0 ? head_dim : 0) * sizeof(float);
}

extern "C" int fmlm_qk_rope_fwd(const fmlm_qk_rope_args* a, void* stream) { return fmlm::run(a, false, stream); }

extern "C" int fmlm_qk_rope_bwd(const fmlm_qk_rope_args* a, void* stream) { return fmlm::run(a, true, stream); }
