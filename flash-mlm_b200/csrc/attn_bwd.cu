// C-ABI entry point of the attention backward pass: argument checks, tensor
// maps and the launches (row statistics, float16: ranges by sequence, Q pass, KV pass).
#include <cmath>
#include <type_traits>

#include "common.h"
#include "tma_map.h"

#include "attn_bwd.cuh"

namespace fmlm {
namespace {

constexpr unsigned long long kTimeoutNs = 2000000000ull;  // 2 s per wait
constexpr size_t kCounterBytes = 256;

template <int D, bool KV, bool BF16>
int launch_pass(const CUtensorMap* m, const BwdParams& p, cudaStream_t s) {
  using C = BwdCfg<D, KV>;
  auto kern = attn_bwd_kernel<D, KV, BF16>;
  // One CTA per SM: a second one would block in tcgen05.alloc.
  const int smem = std::max(C::SMEM_BYTES, 116 * 1024);
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(FMLM_ERR_CUDA, "device ordinal %d out of range", dev);
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return set_error(FMLM_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  kern<<<std::min(p.num_items, device_sm_count()), C::THREADS, smem, s>>>(m[0], m[1], m[2], m[3], m[4], m[5], p);
  return check_launch("attn_bwd_kernel");
}

template <int D, bool KV, bool BF16>
int run_pass(const CUtensorMap* m, BwdParams p, cudaStream_t s) {
  using C = BwdCfg<D, KV>;
  const long long items = (long long)(KV ? p.HK : p.H) * (p.slots + (KV ? p.cslots : 0)) * C::NDH;
  if (items > 0x7fff0000LL) return set_error(FMLM_ERR_INVALID, "problem too large");
  if (items == 0) return FMLM_OK;
  p.num_items = (int)items;
  p.counter += KV ? 1 : 0;
  return launch_pass<D, KV, BF16>(m, p, s);
}

// Tensor maps of q, dout, k, v and the context's k, v with boxes of qrows / krows rows.
int encode_maps(CUtensorMap* m, const fmlm_attn_bwd_args* a, bool ctx, int qrows, int krows) {
  const int D = a->head_dim;
  int rc;
  if ((rc = encode_view(&m[0], a->q, D, qrows, a->dtype, a->q.data, "q"))) return rc;
  if ((rc = encode_view(&m[1], a->dout, D, qrows, a->dtype, a->q.data, "dout"))) return rc;
  if ((rc = encode_view(&m[2], a->k, D, krows, a->dtype, a->q.data, "k"))) return rc;
  if ((rc = encode_view(&m[3], a->v, D, krows, a->dtype, a->q.data, "v"))) return rc;
  if (!ctx) {  // never loaded from
    m[4] = m[2];
    m[5] = m[3];
    return FMLM_OK;
  }
  if ((rc = encode_view(&m[4], a->k_context, D, krows, a->dtype, a->q.data, "k_context"))) return rc;
  return encode_view(&m[5], a->v_context, D, krows, a->dtype, a->q.data, "v_context");
}

template <int D, bool BF16>
int run_bwd(const fmlm_attn_bwd_args* a, const BwdParams& p, float ext_mul, cudaStream_t s) {
  using C = BwdCfg<D, false>;
  // Tile slots of the statistics (float16: of v's heads too) and of the context's
  // v; a block takes several where they are many and short.
  const long long slots = (long long)(BF16 ? p.H : p.H + p.HK) * p.slots, cslots = (long long)p.HK * p.cslots;
  const long long many = (long long)device_sm_count() * 16;
  const bool packed = a->layout == FMLM_BWD_PACKED;
  const bool short_q = slots >= many && (packed ? p.T / p.slots : std::min(p.N, 128)) <= 32;
  const bool short_c = cslots >= many && p.Tc / p.cslots <= 32;
  const long long gather = ((long long)(p.H + p.HK) * p.B + 3) / 4;
  if (slots > 0x7fffffffLL || cslots + gather > 0x7fffffffLL) return set_error(FMLM_ERR_INVALID, "problem too large");
  // Every map before the first launch: a refused view leaves nothing half done.
  const bool ctx = p.C > 0;
  CUtensorMap m[12];
  int rc = encode_maps(m, a, ctx, C::BM, C::BN);
  if (!rc && C::BM != C::BN) rc = encode_maps(m + 6, a, ctx, C::BN, C::BM);
  if (rc) return rc;
  auto lay = [](const fmlm_view4& v) {
    return BwdRows{reinterpret_cast<const uint16_t*>(v.data), v.batch_stride, v.head_stride, v.row_stride};
  };
  auto stats = [&](auto per_block) {
    constexpr int K = decltype(per_block)::value;
    attn_bwd_stats_kernel<D, BF16, K><<<(unsigned)((slots + K - 1) / K), 256, 0, s>>>(
        p, reinterpret_cast<const uint4*>(a->out), reinterpret_cast<const uint4*>(a->dout.data), a->lse, ext_mul, lay(a->v));
  };
  if (short_q) stats(std::integral_constant<int, 8>());
  else stats(std::integral_constant<int, 1>());
  rc = check_launch("attn_bwd_stats_kernel");
  if constexpr (!BF16) {
    if (!rc && range_by_sequence(p)) {
      auto range = [&](auto per_block) {
        constexpr int K = decltype(per_block)::value;
        const long long cblocks = (cslots + K - 1) / K;
        attn_bwd_range_kernel<D, K><<<(unsigned)(cblocks + gather), 128, 0, s>>>(p, lay(a->v_context), (int)cblocks);
      };
      if (short_c) range(std::integral_constant<int, 4>());
      else range(std::integral_constant<int, 1>());
      rc = check_launch("attn_bwd_range_kernel");
    }
  }
  // Without dq the Q pass still leaves short rows' delta for the KV pass (where
  // there can be such rows).
  if (!rc && (a->dq || a->layout != FMLM_BWD_DENSE || a->seq_len <= C::BN)) rc = run_pass<D, false, BF16>(m, p, s);
  if (!rc && a->dk) rc = run_pass<D, true, BF16>(C::BM != C::BN ? m + 6 : m, p, s);
  return rc;
}

template <bool BF16>
int dispatch_bwd(const fmlm_attn_bwd_args* a, const BwdParams& p, float ext_mul, cudaStream_t s) {
  switch (a->head_dim) {
    case 16: return run_bwd<16, BF16>(a, p, ext_mul, s);
    case 32: return run_bwd<32, BF16>(a, p, ext_mul, s);
    case 64: return run_bwd<64, BF16>(a, p, ext_mul, s);
    case 128: return run_bwd<128, BF16>(a, p, ext_mul, s);
    case 256: return run_bwd<256, BF16>(a, p, ext_mul, s);
    default: return set_error(FMLM_ERR_UNSUPPORTED, "HEAD_DIM must be one of {16, 32, 64, 128, 256}");
  }
}

bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }

int check_view(const fmlm_view4& v, const char* name, int64_t rows, int64_t heads, int64_t batch) {
  if (!v.data) return set_error(FMLM_ERR_INVALID, "%s is required", name);
  if (v.rows != rows || v.heads != heads || v.batch != batch)
    return set_error(FMLM_ERR_INVALID, "%s: the view must be [%lld][%lld][%lld][head_dim]", name, (long long)batch,
                     (long long)heads, (long long)rows);
  return FMLM_OK;
}

}  // namespace
}  // namespace fmlm

using namespace fmlm;

extern "C" size_t fmlm_attn_bwd_workspace_bytes(int64_t rows) {
  return kCounterBytes + (size_t)(rows > 0 ? rows : 0) * (sizeof(float2) + sizeof(uint4) + sizeof(int4));
}

extern "C" int fmlm_attn_bwd(const fmlm_attn_bwd_args* a, void* stream) {
  if (!a) return set_error(FMLM_ERR_INVALID, "null args");
  if (a->dtype != FMLM_DTYPE_F16 && a->dtype != FMLM_DTYPE_BF16) return set_error(FMLM_ERR_INVALID, "dtype must be f16 or bf16");
  const int D = a->head_dim;
  const bool packed = a->layout == FMLM_BWD_PACKED;
  if (a->layout < FMLM_BWD_DENSE || a->layout > FMLM_BWD_PACKED) return set_error(FMLM_ERR_INVALID, "bad layout");
  if (a->batch < 1 || a->num_heads < 1 || a->kv_heads < 1 || a->num_heads % a->kv_heads != 0)
    return set_error(FMLM_ERR_INVALID, "batch, num_heads, kv_heads must be >= 1 and num_heads a multiple of kv_heads");
  if (!packed && (a->seq_len < 1 || a->seq_len > 0x3fffff00)) return set_error(FMLM_ERR_INVALID, "seq_len must be in [1, 2^30)");
  if (packed && (a->total_q_len < 1 || a->total_q_len > 0x3fffff00LL))
    return set_error(FMLM_ERR_INVALID, "total_q_len must be in [1, 2^30)");
  if (!packed && (a->causal_query_seq_attn || a->context_entries))
    return set_error(FMLM_ERR_INVALID, "causal_query_seq_attn and a context need the packed layout");
  if (a->layout != FMLM_BWD_DENSE && !a->cu_seqlens_q) return set_error(FMLM_ERR_INVALID, "cu_seqlens_q is required");
  if (a->context_entries != 0 && a->context_entries != 1 && a->context_entries != a->batch)
    return set_error(FMLM_ERR_INVALID, "context_entries must be 0, 1 or batch");
  if (!a->error_word) return set_error(FMLM_ERR_INVALID, "error_word is required");
  const int64_t qr = packed ? a->total_q_len : a->seq_len, qb = packed ? 1 : a->batch;
  int rc;
  if ((rc = check_view(a->q, "q", qr, a->num_heads, qb))) return rc;
  if ((rc = check_view(a->dout, "dout", qr, a->num_heads, qb))) return rc;
  if ((rc = check_view(a->k, "k", qr, a->kv_heads, qb))) return rc;
  if ((rc = check_view(a->v, "v", qr, a->kv_heads, qb))) return rc;
  // (a stride along an axis of one says nothing: torch leaves any there)
  if ((qr > 1 && a->dout.row_stride != D) || (a->num_heads > 1 && a->dout.head_stride != qr * D) ||
      (qb > 1 && a->dout.batch_stride != a->num_heads * qr * D))
    return set_error(FMLM_ERR_INVALID, "dout must be contiguous");
  const bool ctx = a->context_entries > 0 && a->total_context_len > 0;
  if (ctx) {
    if (a->total_context_len > 0x3fffff00LL) return set_error(FMLM_ERR_INVALID, "total_context_len must be < 2^30");
    if (!a->cu_seqlens_context || (a->dk && (!a->dk_context || !a->dv_context)))
      return set_error(FMLM_ERR_INVALID, "a context needs cu_seqlens_context, and dk_context and dv_context with dk");
    if ((rc = check_view(a->k_context, "k_context", a->total_context_len, a->kv_heads, 1))) return rc;
    if ((rc = check_view(a->v_context, "v_context", a->total_context_len, a->kv_heads, 1))) return rc;
    if (!aligned32(a->dk_context) || !aligned32(a->dv_context))
      return set_error(FMLM_ERR_INVALID, "dk_context and dv_context must be 32-byte aligned");
  }
  if ((a->dk == nullptr) != (a->dv == nullptr) || (!a->dq && !a->dk))
    return set_error(FMLM_ERR_INVALID, "give dq, or dk and dv, or all three");
  if (!a->out || !a->lse || !aligned16(a->out) || !aligned16(a->dout.data))
    return set_error(FMLM_ERR_INVALID, "out and lse are required; out and dout must be 16-byte aligned");
  if (!aligned32(a->dq) || !aligned32(a->dk) || !aligned32(a->dv))
    return set_error(FMLM_ERR_INVALID, "dq, dk, dv must be 32-byte aligned");
  // float16: lse in units of q k^T has to fit the float16 columns (the KV pass
  // reports a row's that does not); a smaller scale would shift log(keys) out.
  const bool bf16 = a->dtype == FMLM_DTYPE_BF16;
  const float mag = std::fabs(a->scale);
  if (!(mag <= (bf16 ? 0x1p64f : 0x1p20f)) || (!bf16 && mag < 0x1p-24f))
    return set_error(FMLM_ERR_INVALID, "scale must be finite, at most 2^64 in magnitude, for float16 in [2^-24, 2^20]");
  const int64_t rows = qb * a->num_heads * qr;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < fmlm_attn_bwd_workspace_bytes(rows))
    return set_error(FMLM_ERR_INVALID, "workspace too small (%zu bytes needed)", fmlm_attn_bwd_workspace_bytes(rows));

  BwdParams p{};
  p.layout = a->layout;
  p.B = a->batch;
  p.H = a->num_heads;
  p.HK = a->kv_heads;
  p.G = a->num_heads / a->kv_heads;
  p.N = a->seq_len;
  p.T = packed ? (int)a->total_q_len : 0;
  p.C = ctx ? a->context_entries : 0;
  p.Tc = ctx ? (int)a->total_context_len : 0;
  p.causal = a->causal_query_seq_attn;
  const long long slots = packed ? p.T / 128 + p.B : (long long)p.B * ((p.N + 127) / 128);
  if (slots > 0x3fffffffLL) return set_error(FMLM_ERR_INVALID, "problem too large");
  p.slots = (int)slots;
  p.cslots = p.C > 0 ? p.Tc / 128 + p.C : 0;
  p.cu_q = a->cu_seqlens_q;
  p.cu_c = a->cu_seqlens_context;
  p.counter = reinterpret_cast<int*>(a->workspace);
  p.xstats = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a->workspace) + kCounterBytes);
  p.range = reinterpret_cast<int4*>(p.xstats + rows);
  p.stats = reinterpret_cast<const float2*>(p.range + rows);
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.dkc = a->dk_context;
  p.dvc = a->dv_context;
  p.scale = a->scale;
  // The exponent's scale, kept away from 0: the KV pass divides lse by it.  At
  // 2^-100 no bfloat16 score moves the exponent; float16's range ends earlier,
  // and its scales are refused above instead.
  const float sl2 = a->scale * 1.4426950408889634f;
  p.scale_log2 = std::fabs(sl2) < 0x1p-100f ? 0x1p-100f : sl2;
  // bfloat16: a power of two near 1 / scale_log2, so that what the columns hold
  // is of lse's own magnitude.  float16's columns have their units.
  p.ext_unit = bf16 ? std::ldexp(1.f, std::min(100, std::max(-100, -std::ilogb(p.scale_log2)))) : 1.f;
  const float ext_mul = 1.f / (p.scale_log2 * p.ext_unit);
  // -400 in the exponent; at float16's smallest scales what the columns hold unsaturated, -92 or less
  p.none = bf16 ? -400.f * ext_mul : std::copysign(std::min(400.f * std::fabs(ext_mul), 0x1p30f), -ext_mul);
  p.err = a->error_word;
  p.timeout_ns = kTimeoutNs;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return bf16 ? dispatch_bwd<true>(a, p, ext_mul, s) : dispatch_bwd<false>(a, p, ext_mul, s);
}
