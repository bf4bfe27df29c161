// Backward pass of the bidirectional attention for sm_100a (B200).
//
// With S = scale * q k^T, P = exp(S - lse) (lse saved by the forward pass),
// dP = dO v^T and delta = rowsum(dO * O):
//   dS = P * (dP - delta),  dV = P^T dO,  dQ = scale * dS k,  dK = scale * dS^T q.
// The probabilities are recomputed tile by tile; nothing of size Nq x Nkv is
// stored.  Two passes over the score tiles, each owning its outputs, so no
// floating-point atomics are needed and the same inputs give the same bits:
//   KV pass  a work item owns 128 keys of one key head; the queries that see
//            them (of every query head of the group) stream past; dK and dV
//            accumulate in TMEM.
//   Q pass   a work item owns 128 queries; their keys stream past (context,
//            then main); dQ accumulates in TMEM.
// Both are one kernel: stationary tiles A1, A2 (128 rows), streamed tiles B1, B2:
//   S = A1 B1^T,  dP = A2 B2^T            (KV: A = K, V; B = Q, dO.  Q: A = Q, dO; B = K, V)
//   acc2 += dS B1,  KV: acc1 += P B2      (P, dS: 16-bit, A operand from TMEM)
// In the KV pass S and dP are the transposed scores, so P^T and dS^T leave the
// registers in the layout in which the tensor cores read A from TMEM, as in
// the Q pass; P and dS never touch shared memory.  lse and delta then belong
// to columns: every thread would have to read all of them from shared memory,
// 128 KB per tile through a 128-byte-a-cycle port (measured: 1800 + 1800 cycles
// a tile for P and dS against 1000 + 650 in the Q pass).  Instead one more K
// step of the score MMAs adds them: B gets 16 more columns that hold -lse (in
// units of the scores) and -delta as sums of three or four 16-bit numbers, A
// the units of these, so S and dP arrive with them subtracted (ext_columns).
//
// delta is dO * O with O as the forward pass returned it, in 16 bits.  Over many
// keys that costs little (dq, dk within 1.5 of the error of gradients that are
// only rounded at the end), but not over a few, where O is as large as v: two
// keys, 2.4.  So a Q item whose keys fit one tile (or are at most 64 in two
// ranges, which it then walks twice) sums delta = sum_k P dP itself, in 32 bits
// (1.4), and leaves it for the KV pass, which runs after.  Rows of many keys
// whose probability lies on a few keep O's rounding (2.2 at scores of deviation 3).
//
// P and dS are rounded to 16 bits for the tensor cores, half a step of each
// term: next to the rounding of the result that is a factor of 1.4 in a
// gradient's error when many terms average it, and up to 2 when there are few.
// So items that stream few rows, or hold the few rows of a short sequence, give
// P and dS as the sum of two 16-bit numbers, the second in the TMEM columns
// that the first leaves free, for another K walk of the accumulating MMAs
// (factor 1.0; all items that way would add 2 to the 7 matrix products).
//
// float16 P is held times 2^12 (P <= 1), and dS times a power of two that brings
// its bound |dO| |v| + |delta| to 2^15: as it is, dS of long rows or of small dO
// would lie among float16's subnormals (4096 keys, dO of 1e-3: dq and dk 8 times
// as far off as gradients rounded once, now 1.1), and dS of large dO past its
// end.  A Q item's rows have each their own power, from the row's dO and the
// largest v that it sees; a KV item one, from its sequence's v and the dO and
// delta that stream past.  The statistics kernel leaves each tile's largest, so
// that none depends on rows it does not see.
//
// What bounds it: the tensor pipe at head_dim 128 (16 heads of 8192 tokens,
// bf16: Q pass 629 us, 1310 TFLOP/s; KV pass 728 us, 1511 TFLOP/s, 70 % of the
// tensor cycles), the chain exponentials - TMEM - MMA at head_dim 64 (2 x 16
// heads of 2048 tokens: 76 and 90 us, tensor pipe 40 and 52 %, exponentials'
// unit 53 and 46 %).
//
// Roles of a persistent CTA (one per SM): warps 0-15 do the element-wise work
// (warp w: TMEM lanes 32 (w % 4) .., column quarter w / 4 of every score tile),
// warp 16 loads tiles by TMA and decodes work items, warp 17 issues the MMAs,
// warp 18 (KV) copies the streamed rows' extra columns, warps 18 (items of one
// tile) and 19 (KV, float16) find dS's power of two.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace fmlm {

constexpr int kErrStatistics = 7;

struct BwdParams {
  int layout;  // FMLM_BWD_*
  int B, H, HK, G, N;
  int T, Tc;   // packed rows per head; context rows per head
  int C;       // context entries (0: none)
  int causal;
  int slots, cslots;  // tile slots of a head over the sequences / context entries
  int num_items;
  const int* cu_q;
  const int* cu_c;
  const float2* stats;  // per output row: {-lse * log2(e) + kPExp, -delta}
  uint4* xstats;        // the same as what the KV pass puts into B's extra columns; float16: with the code
                        // (mag_code) of |dO| in the last column, whose unit is 0
  int4* range;          // float16: the codes of a tile's largest |dO|, |delta| (x, y: at the tile's first row of the
                        // query head) and |v| (z: of the key head); at a sequence's first row, where
                        // range_by_sequence, all its tiles' (and in z, times 256, that of all sequences up to it)
                        // and its context's |v| (w; a shared context's at row 0)
  float none;           // KV: -lse, as the columns hold it, of a row that is not there: P = 0
  int* counter;
  void *dq, *dk, *dv, *dkc, *dvc;
  float scale, scale_log2;  // scale_log2: of the scores in the exponent (never 0: see the host code)
  float ext_unit;           // KV, bfloat16: unit (a power of two) of the lse columns
  int* err;
  unsigned long long timeout_ns;
};

template <int D_, bool KV_>
struct BwdCfg {
  static constexpr int D = D_;
  static constexpr bool KV = KV_;
  static constexpr int BM = 128;
  static constexpr int BN = D == 256 ? 64 : 128;  // streamed rows per tile (D = 256: what shared memory holds)
  // D = 256: dK and dV of 128 keys (512 fp32 columns) would fill TMEM, so a KV
  // item makes one 128-column half of both and the scores are computed twice.
  static constexpr int DV = (KV && D == 256) ? 128 : D;
  static constexpr int NDH = D / DV;
  static constexpr int SWB = D * 2 >= 128 ? 128 : D * 2;
  static constexpr int SLAB_COLS = SWB / 2;
  static constexpr int NSLAB = D / SLAB_COLS;
  static constexpr int A_BYTES = BM * D * 2;
  static constexpr int B_BYTES = BN * D * 2;
  static constexpr int STAGES = D <= 64 ? 4 : D == 128 ? 2 : 1;
  // The stationary tiles as A operands in TMEM, where there is room: with both
  // operands in shared memory an MMA of 128 x 128 x 16 reads 8 KB in 64 cycles,
  // all that shared memory delivers, and every barrier and load waits behind it.
  static constexpr bool ATM = KV ? D <= 64 : D <= 128;
  // P in columns of its own (KV): the next S need not wait until P is consumed.
  static constexpr bool SEP_P = KV && D <= 64;
  // P and dS over S and dP (D = 128): each is handed over in two halves, 16 of
  // a warp's 32 columns at a time, so that the MMAs of the first half run while
  // the second is computed.  What waits for them (the next S, the next dP)
  // starts that much earlier (8192 tokens: KV pass 759 -> 726 us; the Q pass,
  // where only dP waits, gained nothing).
  static constexpr bool SPLIT = KV && D == 128;
  // Two buffers of dP / dS (Q, where TMEM has the columns): the next dP is
  // issued with the next S instead of behind this tile's accumulation (head_dim
  // 64, a shared context of 1024 keys: Q pass 136 -> 130 us; with earlier
  // sequences 425 -> 405).
  static constexpr bool DB = !KV && D <= 64;
  static constexpr int EW_GROUPS = 4;
  static constexpr int EW_WARPS = 4 * EW_GROUPS;
  static constexpr int TMA_WARP = EW_WARPS;
  static constexpr int MMA_WARP = EW_WARPS + 1;
  static constexpr int EXT_WARP = EW_WARPS + 2;
  static constexpr int POWER_WARP = EW_WARPS + 3;  // (float16; registers are given to four warps at a time)
  static constexpr int THREADS = 32 * (EW_WARPS + (KV ? 4 : 2));
  static constexpr int NC = BN / EW_GROUPS;  // score columns per element-wise warp
  static constexpr int TM_S = 0, TM_DP = BN, TM_P = SEP_P ? 2 * BN : 0;
  static constexpr int TM_ACC1 = (DB ? 3 : 2) * BN + (SEP_P ? BN / 2 : 0), TM_ACC2 = TM_ACC1 + (KV ? DV : 0);
  static constexpr int TM_A1 = TM_ACC2 + DV, TM_A2 = TM_A1 + (ATM ? D / 2 : 0);
  static constexpr int TMEM_USED = TM_A2 + (ATM ? D / 2 : 0);
  static_assert(TMEM_USED <= 512, "TMEM budget");
  static constexpr int TMEM_COLS = TMEM_USED <= 256 ? 256 : 512;
  // KV: the extra K step, 32-byte rows: A's constants, and per stage B1's and B2's columns
  static constexpr int AX_BYTES = KV ? BM * 32 : 0;
  static constexpr int BX_BYTES = KV ? BN * 32 : 0;
  static constexpr int SMEM_TILES = 2 * A_BYTES + 2 * STAGES * B_BYTES + AX_BYTES + 2 * STAGES * BX_BYTES;
  static constexpr int SUM_BYTES = KV ? 0 : 2 * EW_GROUPS * BM * 4;  // Q: delta's partial sums, twice
  static constexpr int EXACT_KEYS = 64;  // Q: items of several tiles with at most so many keys sum delta themselves
  static constexpr int FEW_TERMS = 128, FEW_ROWS = 8;  // items whose P and dS keep a second part (see above)
  static constexpr int RING = 4;
  static constexpr int ITEM_BYTES = 104;
  static constexpr int SMEM_BYTES = SMEM_TILES + 512 + RING * ITEM_BYTES + SUM_BYTES + 1024;
};

// A work item: the stationary tile, the rows it writes and up to two ranges of
// streamed rows (the KV pass walks its one range once per query head of the group).
struct BwdItem {
  int a_map, a_row, a_h, a_b;  // stationary tile: 0 main tensors, 1 context; coordinates
  int valid, limit;            // rows [0, valid) hold results, [valid, limit) get zeros
  int dh;                      // D = 256 KV pass: 128-column half
  int heads, h0, b;            // streamed heads h0 .. h0 + heads - 1, batch coordinate
  int map0, row0, end0, nt0;   // first range (context when map0 = 1)
  int row1, end1, nt1;         // second range (main)
  int stat_h;                  // KV: stats rows of one streamed head
  int pre;                     // Q: tiles walked first for delta alone (0 or all of them)
  int few;                     // few terms or few rows: P and dS keep a second 16-bit part
  int seq;                     // sequence, or context entry
  float ds_mul;                // KV, float16: what takes P (dP - delta) to the dS that is held
  long long out_row;           // output row of the tile's row 0 (also its stats row in the Q pass)
  long long stat0;             // KV: stats row of (head h0, streamed row 0)
};
static_assert(sizeof(BwdItem) <= 104, "item ring slot");

// The sequence that owns tile slot v when sequence b's tiles start at slot
// cu[b] / 128 + b (strictly increasing, and at least ceil(len / 128) apart, so
// no scan is needed).  A 32-way search by the whole warp.
__device__ __forceinline__ int find_slot_owner(const int* __restrict__ cu, int n, int v, int lane) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int i = lo + lane * step;
    const bool le = i < hi && (lane == 0 || ((__ldg(cu + i) >> 7) + i) <= v);
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int top = 31 - __clz(m);
    lo += top * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Magnitudes as small whole numbers: 64 + X where the value is below 2^X (and
// not below 2^(X - 2)), 0 of a 0, at most 126 (infinities).
__device__ __forceinline__ int mag_code(float x) {  // x >= 0
  return x > 0.f ? min(max(((__float_as_int(x) >> 23) & 255) - 126 + 64, 1), 126) : 0;
}
__device__ __forceinline__ int mag_code_of_square(float x) {
  return x > 0.f ? min(max(((((__float_as_int(x) >> 23) & 255) - 125) >> 1) + 64, 1), 126) : 0;
}
// The power of two for dS = P (dP - delta) from the codes of |dO|, |v| and |delta|:
// |dS| 2^power <= 2^15, half of what float16 holds.  But dS is made smaller only
// for the sake of |dO|, as if |v| were 32 at most: one far larger row of v would
// push the others' dS among the subnormals, though nothing may attend to it.
__device__ __forceinline__ int ds_power(int g, int v, int d) {
  const int bound = max(g > 0 && v > 0 ? g + v - 64 : 0, d) - 64 + 1;
  const int least = min(0, 15 - (g - 64 + 5 + 1));
  return min(max(15 - bound, least), 60);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ float inv_pow2(float x) { return __int_as_float((254 << 23) - __float_as_int(x)); }  // x = 2^e

// Rows [s0, s1) of sequence b in a packed batch.
__device__ __forceinline__ void packed_rows(const BwdParams& p, int b, int& s0, int& s1) {
  s0 = min(max(__ldg(p.cu_q + b), 0), p.T);
  s1 = min(max(__ldg(p.cu_q + b + 1), 0), p.T);
}

// Items that see several sequences would read many tiles' codes: another kernel
// gathers each sequence's at its first row (64 sequences of 32 to 256 tokens, each
// seeing the earlier ones and a context: Q 417 -> 406, KV 625 -> 620 us).
__host__ __device__ __forceinline__ bool range_by_sequence(const BwdParams& p) { return p.C > 0 || p.causal; }

// KV: whether the rows that stream past are of several sequences.
__device__ __forceinline__ bool streams_several(const BwdParams& p, const BwdItem& it) {
  return it.a_map ? p.C == 1 : p.causal != 0;
}

// KV: the code of the largest |v| of an item's keys (a context's: of its entry).
__device__ __forceinline__ int kv_item_value_code(const BwdParams& p, const BwdItem& it) {
  if (it.a_map) return __ldg(&p.range[(long long)it.a_h * p.T + (p.C == 1 ? 0 : it.row0)].w);
  return __ldg(&p.range[it.out_row].z) & 255;
}

// KV: dS's power of two for an item, by the whole warp.
__device__ __forceinline__ int kv_item_power(const BwdParams& p, const BwdItem& it, bool several, int lane) {
  const int v = kv_item_value_code(p, it), heads = it.heads;
  const int4* range = p.range + it.stat0;
  int g = 0, d = 0;
  auto take = [&](const int4* x) {
    const int2 c = __ldg(reinterpret_cast<const int2*>(x));
    g = max(g, c.x);
    d = max(d, c.y);
  };
  if (!several) {
    const int k = range_by_sequence(p) ? 1 : (it.end0 - it.row0 + 127) >> 7;  // a head's
    for (int i = lane; i < k * heads; i += 32) {
      const int h = heads == 1 ? 0 : i / k;
      take(range + (long long)h * it.stat_h + it.row0 + (i - h * k) * 128);
    }
  } else {  // all sequences (of a shared context), or those from the item's on
    const int b0 = it.a_map ? 0 : it.seq, nb = p.B - b0;
    for (int i = lane; i < nb * heads; i += 32) {
      const int h = heads == 1 ? 0 : i / nb;
      int s0, s1;
      packed_rows(p, b0 + i - h * nb, s0, s1);
      if (s1 > s0) take(range + (long long)h * it.stat_h + s0);
    }
  }
  return ds_power(__reduce_max_sync(0xffffffffu, g), v, __reduce_max_sync(0xffffffffu, d));
}

// Q: the code of the largest |v| that an item's rows see, by the whole warp.
__device__ __forceinline__ int q_item_value_code(const BwdParams& p, const BwdItem& it, int lane) {
  const bool packed = p.layout == FMLM_BWD_PACKED;
  const int r0 = !packed ? 0 : p.causal ? min(max(__ldg(p.cu_q + it.seq), 0), p.T) : p.C > 0 ? it.row1 : it.row0;
  const int4* at = p.range + ((packed ? (long long)it.h0 * p.T : ((long long)it.b * p.HK + it.h0) * p.N) + r0);
  int v = 0;
  if (range_by_sequence(p)) {
    const int2 c = __ldg(reinterpret_cast<const int2*>(&at->z));
    v = p.causal ? c.x >> 8 : c.x & 255;
    if (p.C > 0) v = max(v, p.C == 1 ? __ldg(&p.range[(long long)it.h0 * p.T].w) : c.y);
    return v;
  }
  for (int t = lane * 128; t < it.end0 - r0; t += 32 * 128) v = max(v, __ldg(&at[t].z) & 255);
  return __reduce_max_sync(0xffffffffu, v);
}

template <class C>
__device__ __forceinline__ BwdItem decode_bwd_item(const BwdParams& p, int w, int lane) {
  BwdItem it;
  constexpr int BN = C::BN;
  auto tiles = [](int r0, int r1) { return r1 > r0 ? (r1 - r0 + BN - 1) / BN : 0; };
  it.dh = w % C::NDH;
  w /= C::NDH;
  // Heads fastest, and the longest items first, so that none is left for the
  // end: the context's (a shared one streams the whole batch past) before the
  // sequences', and with causal_query_seq_attn the sequences with most to
  // stream (KV pass: the first, Q pass: the last) before the others.
  // Sequences of one length (dense) go head by head instead, whose streamed
  // tiles then stay in L2 (16 heads of 8192 x 128: KV 793 -> 768, Q 649 -> 628 us).
  const int heads = C::KV ? p.HK : p.H;
  const bool dense = p.layout == FMLM_BWD_DENSE;
  const int h = dense ? w / p.slots : w % heads;
  int v = dense ? w % p.slots : w / heads;
  const bool ctx = C::KV && v < p.cslots;
  if (C::KV && !ctx) v -= p.cslots;
  if (!C::KV && p.causal) v = p.slots - 1 - v;
  const bool packed = p.layout == FMLM_BWD_PACKED;
  it.map0 = 0; it.row1 = it.end1 = it.nt1 = 0;
  it.a_map = ctx ? 1 : 0;
  it.a_h = h;
  it.a_b = it.b = 0;
  it.heads = C::KV ? p.G : 1;
  it.h0 = C::KV ? h * p.G : h / p.G;
  it.stat_h = 0;
  it.stat0 = 0;
  int tile = 0;  // of its sequence
  if (ctx) {
    const int c = it.seq = find_slot_owner(p.cu_c, p.C, v, lane);
    const int c0 = min(max(__ldg(p.cu_c + c), 0), p.Tc), c1 = min(max(__ldg(p.cu_c + c + 1), 0), p.Tc);
    const int t = tile = v - ((c0 >> 7) + c);
    it.a_row = c0 + t * 128;
    it.valid = it.limit = min(max(c1 - it.a_row, 0), t >= 0 ? 128 : 0);
    it.out_row = (long long)h * p.Tc + it.a_row;
    const int e = p.C == 1 ? p.B : c + 1;
    it.row0 = min(max(__ldg(p.cu_q + (p.C == 1 ? 0 : c)), 0), p.T);
    it.end0 = min(max(__ldg(p.cu_q + e), 0), p.T);
    it.stat_h = p.T;
  } else if (packed) {
    const int b = it.seq = find_slot_owner(p.cu_q, p.B, v, lane);
    int s0, s1;
    packed_rows(p, b, s0, s1);
    const int t = tile = v - ((s0 >> 7) + b);
    it.a_row = s0 + t * 128;
    it.valid = it.limit = min(max(s1 - it.a_row, 0), t >= 0 ? 128 : 0);
    it.out_row = (long long)h * p.T + it.a_row;
    it.stat_h = p.T;
    it.row0 = s0;
    it.end0 = s1;
    if (C::KV && p.causal) it.end0 = min(max(__ldg(p.cu_q + p.B), 0), p.T);
    if (!C::KV) {
      if (p.causal) it.row0 = 0;
      if (p.C > 0) {  // context first, then main
        const int c = p.C == 1 ? 0 : b;
        it.row1 = it.row0; it.end1 = it.end0;
        it.nt1 = tiles(it.row1, it.end1);
        it.map0 = 1;
        it.row0 = min(max(__ldg(p.cu_c + c), 0), p.Tc);
        it.end0 = min(max(__ldg(p.cu_c + c + 1), 0), p.Tc);
      }
    }
  } else {
    const int per_seq = (p.N + 127) / 128;
    const int b = v / per_seq, t = v % per_seq;
    int L = p.N;
    if (p.layout == FMLM_BWD_PADDED) L = min(max(__ldg(p.cu_q + b + 1) - __ldg(p.cu_q + b), 0), p.N);
    it.seq = b;
    tile = t;
    it.a_row = t * 128;
    it.a_b = it.b = b;
    it.valid = min(max(L - it.a_row, 0), 128);
    it.limit = min(p.N - it.a_row, 128);
    it.out_row = ((long long)b * (C::KV ? p.HK : p.H) + h) * p.N + it.a_row;
    it.row0 = 0;
    it.end0 = L;
    it.stat_h = p.N;
  }
  if (C::KV) it.stat0 = ((long long)(packed ? 0 : it.b) * p.H + it.h0) * it.stat_h;
  it.nt0 = tiles(it.row0, it.end0);
  if (it.valid == 0) it.nt0 = it.nt1 = 0;
  it.pre = 0;
  it.ds_mul = 0.f;
  const int n = it.nt0 + it.nt1, terms = max(it.end0 - it.row0, 0) + max(it.end1 - it.row1, 0);
  it.few = (it.valid <= C::FEW_ROWS && tile == 0) || (long long)it.heads * terms <= C::FEW_TERMS;
  if constexpr (!C::KV) {
    if (n > 1 && terms <= C::EXACT_KEYS) it.pre = n;
    if (n == 1 || it.pre > 0) it.few = 1;
    // dq not asked for: only items that have a delta to leave
    if (p.dq == nullptr && n != 1 && it.pre == 0) it.valid = it.limit = it.nt0 = it.nt1 = 0;
  }
  return it;
}

struct __align__(8) BwdBarriers {
  uint64_t a_full, a_empty;
  uint64_t b1_full[4], b2_full[4], b1_empty[4], b2_empty[4];
  uint64_t a_tm;              // element-wise -> MMA: the stationary tiles are in TMEM
  uint64_t s_full, dp_full[2];  // MMA -> element-wise: S / dP (of either buffer) complete
  uint64_t s_free;            // element-wise -> MMA: S is in registers
  uint64_t p_full[2], ds_full[2];  // element-wise -> MMA: P / dS written (its first, second half; or dS in either buffer)
  uint64_t p_free;            // MMA -> element-wise (separate P): P consumed
  uint64_t sum_full;          // Q: every warp's part of delta is in shared memory
  uint64_t acc_full, acc_empty;
  uint64_t item_full[4], item_empty[4];
  uint64_t mul_full[4];       // KV, float16: extra-column or power warp -> element-wise: the item's ds_mul
  int item_idx[4];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(BwdBarriers) <= 512, "barrier block is reserved 512 bytes");

// float16 holds P scaled by 2^12 (P <= 1): small probabilities of long rows
// stay clear of its subnormals.  bfloat16 has the exponent range as it is.
template <bool BF16>
struct BwdScale {
  static constexpr float kPExp = BF16 ? 0.f : 12.f;
  static constexpr float kInv = BF16 ? 1.f : 1.f / 4096.f;
};

// MMA issue with the shared-memory descriptors as (low word, constant high
// word): the low word holds the address, so stepping through a tile is one
// 32-bit add and the high words never leave their registers.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tm, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a_tm), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc)
      : "memory");
}

// Two float32 operations in one instruction (sm_100): the element-wise warps
// are bound by issue slots and the exponentials' unit, not by arithmetic.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2u(uint32_t a, uint32_t b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void unf2(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// One whole 32-byte sector: a thread owns a row, so neighbouring lanes write
// far apart, and half sectors would cost the memory system twice.
__device__ __forceinline__ void st_sector(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// 16-byte vector c of row r of a K-major tile as TMA's swizzle laid it out.
template <int SWB>
__device__ __forceinline__ uint4 ld_swizzled(const uint8_t* tile, int rows, int r, int c) {
  constexpr int V = SWB / 16;  // vectors per row of a slab
  const int x = ((r * SWB) >> 7) & (V - 1);
  return *reinterpret_cast<const uint4*>(tile + (c / V) * (rows * SWB) + r * SWB + (((c % V) ^ x) << 4));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(F2 v) {
  float a, b;
  unf2(v, a, b);
  return pack2<BF16>(a, b);
}

template <bool BF16>
__device__ __forceinline__ F2 unpack2(uint32_t u) {
  if constexpr (BF16) return f2u(u << 16, u & 0xffff0000u);
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u));
  return f2(v.x, v.y);
}

// What rounding v to the pair u left over, as another pair.
template <bool BF16>
__device__ __forceinline__ uint32_t pack_rest(F2 v, uint32_t u) {
  return pack2<BF16>(fma2(unpack2<BF16>(u), f2(-1.f, -1.f), v));
}

// 16-byte half h of row r of a tile of 32-byte rows in the 32-byte swizzle.
__device__ __forceinline__ uint8_t* ext_row(uint8_t* tile, int r, int h) {
  return tile + r * 32 + ((h ^ ((r >> 2) & 1)) << 4);
}

// The extra columns' units (A's constants): four columns of B1 for lse, three
// of B2 for delta.  bfloat16 has float32's exponents, so three numbers of one
// unit hold a value to 2^-27 of it.  float16 has not: its units fall by 2^11
// or 2^12, the bits of one number.  lse, in units of q k^T, fits to 2^-48 of it
// or 2^-39, whichever is larger, up to 65504 * 2^15; delta to 2^-36 of it or
// 2^-37, up to 65504 * 2^12.  What is larger saturates, and the KV pass says so.
template <bool BF16>
__device__ __forceinline__ uint4 ext_units(float bf16_unit) {
  if constexpr (BF16)
    return make_uint4(pack2<BF16>(bf16_unit, bf16_unit), pack2<BF16>(bf16_unit, 0.f), pack2<BF16>(1.f, 1.f), pack2<BF16>(1.f, 0.f));
  else
    return make_uint4(pack2<BF16>(0x1p15f, 0x1p4f), pack2<BF16>(0x1p-7f, 0x1p-14f), pack2<BF16>(0x1p12f, 1.f), pack2<BF16>(0x1p-12f, 0.f));
}

// The float16 number of this unit that v is nearest to, taken off v (exactly).
// Saturates; of infinities and NaN it makes NaN.
__device__ __forceinline__ float take_half(float& v, float unit) {
  const float c = __half2float(__float2half_rn(fminf(fmaxf(v / unit, -65504.f), 65504.f) + (v - v)));
  v = fmaf(-c, unit, v);
  return c;
}

// The extra columns of a row: four of B1 (lse) in x, y; three of B2 (delta) in z, w.
template <bool BF16>
__device__ __forceinline__ uint4 ext_columns(float nl, float nd) {
  float l[4], d[3];
  if constexpr (BF16) {
    auto split3 = [](float v, float* o) {
      o[0] = __bfloat162float(__float2bfloat16_rn(v));
      o[1] = __bfloat162float(__float2bfloat16_rn(v - o[0]));
      o[2] = v - o[0] - o[1];
    };
    split3(nl, l);
    split3(nd, d);
    l[3] = 0.f;
  } else {
    l[0] = take_half(nl, 0x1p15f);
    l[1] = take_half(nl, 0x1p4f);
    l[2] = take_half(nl, 0x1p-7f);
    l[3] = take_half(nl, 0x1p-14f);
    d[0] = take_half(nd, 0x1p12f);
    d[1] = take_half(nd, 1.f);
    d[2] = take_half(nd, 0x1p-12f);
  }
  return make_uint4(pack2<BF16>(l[0], l[1]), pack2<BF16>(l[2], l[3]), pack2<BF16>(d[0], d[1]), pack2<BF16>(d[2], 0.f));
}

// float16: the columns' first numbers are at their end (or past it).
__device__ __forceinline__ bool ext_saturated(const uint4& x) {
  return (x.x & 0x7fffu) == 0x7bffu || (x.z & 0x7fffu) == 0x7bffu;
}

template <int D, bool KV, bool BF16>
__global__ void __launch_bounds__(BwdCfg<D, KV>::THREADS, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ CUtensorMap tm_kc, const __grid_constant__ CUtensorMap tm_vc,
                    const BwdParams p) {
  using C = BwdCfg<D, KV>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  constexpr int BN = C::BN, SWB = C::SWB, STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;                        // [A1, A2]
  uint8_t* sB = sA + 2 * C::A_BYTES;         // [STAGES][B1, B2]
  uint8_t* sAx = sB + 2 * STAGES * C::B_BYTES;  // KV: A's constants of the extra K step
  uint8_t* sBx = sAx + C::AX_BYTES;             // KV: [STAGES][B1's, B2's extra columns]
  BwdBarriers* bar = reinterpret_cast<BwdBarriers*>(smem + C::SMEM_TILES);
  BwdItem* ring_items = reinterpret_cast<BwdItem*>(reinterpret_cast<uint8_t*>(bar) + 512);
  float* sSum = reinterpret_cast<float*>(ring_items + C::RING);  // Q: [2][EW_GROUPS][BM]
  volatile int* abort_flag = &bar->abort_flag;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bar->a_full, 1);
    mbar_init(&bar->a_empty, C::ATM ? C::EW_WARPS : 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar->b1_full[i], KV ? 2 : 1);  // KV: the tile, and its rows' extra columns
      mbar_init(&bar->b2_full[i], 1);
      mbar_init(&bar->b1_empty[i], 1);
      mbar_init(&bar->b2_empty[i], 1);
      mbar_init(&bar->item_full[i], 1);
      mbar_init(&bar->mul_full[i], 1);
      mbar_init(&bar->item_empty[i], C::EW_WARPS + (!KV ? 1 : BF16 ? 2 : 3));
    }
    mbar_init(&bar->s_full, 1);
    mbar_init(&bar->a_tm, C::EW_WARPS);
    mbar_init(&bar->s_free, C::EW_WARPS);
    mbar_init(&bar->p_free, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->dp_full[i], 1);
      mbar_init(&bar->p_full[i], C::EW_WARPS);
      mbar_init(&bar->ds_full[i], C::EW_WARPS);
    }
    mbar_init(&bar->sum_full, C::EW_WARPS);
    mbar_init(&bar->acc_full, 1);
    mbar_init(&bar->acc_empty, C::EW_WARPS);
    bar->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == C::MMA_WARP) {
    tmem_alloc(&bar->tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  if constexpr (KV) {
    // Rows of 32 bytes in the 32-byte swizzle.  A's: the columns' units, then
    // zeros; B's second halves: zeros.
    for (int r = threadIdx.x; r < C::BM; r += C::THREADS) {
      *reinterpret_cast<uint4*>(ext_row(sAx, r, 0)) = ext_units<BF16>(p.ext_unit);
      *reinterpret_cast<uint4*>(ext_row(sAx, r, 1)) = make_uint4(0, 0, 0, 0);
    }
    for (int r = threadIdx.x; r < 2 * STAGES * BN; r += C::THREADS)
      *reinterpret_cast<uint4*>(ext_row(sBx + (r / BN) * C::BX_BYTES, r % BN, 1)) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  if (warp == C::TMA_WARP && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_do);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bar->tmem_base;
  const uint64_t tmo = p.timeout_ns;
  const int num_items = p.num_items;
  bool failed = false;

  auto fail = [&]() {
    failed = true;
    *abort_flag = 1;
    atomicExch(p.err, 1);
  };
  // Whole-warp wait; false once anything in the CTA has given up.
  auto wait_for = [&](uint64_t* b, uint32_t ph, uint64_t limit) -> bool {
    if (__all_sync(0xffffffffu, mbar_try_wait(smem_u32(b), ph))) return true;
    if (!mbar_wait(b, ph, abort_flag, limit)) fail();
    failed = __any_sync(0xffffffffu, failed);
    return !failed;
  };
  auto wait = [&](uint64_t* b, uint32_t ph) -> bool { return wait_for(b, ph, tmo); };
  // The next published item, in its ring slot until release_item; nullptr: no more.
  auto take_item = [&](uint32_t ring, uint64_t limit) -> const BwdItem* {
    if (failed || !wait_for(&bar->item_full[ring & 3], (ring >> 2) & 1u, limit)) return nullptr;
    const int w = *reinterpret_cast<volatile int*>(&bar->item_idx[ring & 3]);
    return w < num_items ? ring_items + (ring & 3) : nullptr;
  };
  auto release_item = [&](uint32_t ring) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar->item_empty[ring & 3]);
  };

  if (warp == C::TMA_WARP) {
    // ------------------------------------------------------------ producer
    uint32_t fill = 0, aload = 0;
    int w = blockIdx.x;
    auto load_tile = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* b, int rows, int row, int h, int bb) {
      for (int s = 0; s < C::NSLAB; ++s) tma_load_4d(dst + s * (rows * SWB), m, b, s * C::SLAB_COLS, row, h, bb);
    };
    // The next item that writes something, decoded (w >= num_items: none).  Its
    // counter and offset loads take some 2000 cycles, so it is fetched before the
    // current item's last tile is; not earlier, since a CTA in a long item
    // would then hold back work that others are free to take (measured: a
    // shared context's items, 72 tiles each, 202 -> 220 us).
    BwdItem it;
    auto fetch = [&](BwdItem& x) {
      for (;;) {
        if (w >= num_items) return;
        x = decode_bwd_item<C>(p, w, lane);
        if (x.limit > 0) return;  // (a slot past its sequence's end writes nothing)
        int next = 0;
        if (lane == 0) next = (int)gridDim.x + atomicAdd(p.counter, 1);
        w = __shfl_sync(0xffffffffu, next, 0);
      }
    };
    fetch(it);
    for (uint32_t ring = 0;; ++ring) {
      if (!wait(&bar->item_empty[ring & 3], ((ring >> 2) & 1u) ^ 1u)) break;
      if (lane == 0) {
        if (w < num_items) ring_items[ring & 3] = it;
        bar->item_idx[ring & 3] = w;
        mbar_arrive(&bar->item_full[ring & 3]);
      }
      __syncwarp();
      if (w >= num_items) break;
      BwdItem nx;
      auto prefetch = [&]() {
        int next = 0;
        if (lane == 0) next = (int)gridDim.x + atomicAdd(p.counter, 1);
        w = __shfl_sync(0xffffffffu, next, 0);
        fetch(nx);
      };
      const int n = it.heads * it.nt0 + it.nt1 + it.pre;
      if (n > 0) {
        if (!wait(&bar->a_empty, (aload & 1u) ^ 1u)) break;
        if (lane == 0) {
          const CUtensorMap* m1 = KV ? (it.a_map ? &tm_kc : &tm_k) : &tm_q;
          const CUtensorMap* m2 = KV ? (it.a_map ? &tm_vc : &tm_v) : &tm_do;
          mbar_arrive_expect_tx(&bar->a_full, 2 * C::A_BYTES);
          load_tile(sA, m1, &bar->a_full, C::BM, it.a_row, it.a_h, it.a_b);
          load_tile(sA + C::A_BYTES, m2, &bar->a_full, C::BM, it.a_row, it.a_h, it.a_b);
        }
        __syncwarp();
        ++aload;
        int g = 0, t = 0;  // streamed head, tile within it (Q pass: tile over both ranges)
        for (int i = 0; i < n && !failed; ++i, ++fill) {
          const int st = fill % STAGES;
          const uint32_t ph = (fill / STAGES) & 1u;
          const bool second = !KV && t >= it.nt0;
          const int row = second ? it.row1 + (t - it.nt0) * BN : it.row0 + t * BN;
          const int h = it.h0 + g;
          const bool cmap = !KV && it.map0 == 1 && !second;
          uint8_t* d1 = sB + st * 2 * C::B_BYTES;
          if (!wait(&bar->b1_empty[st], ph ^ 1u)) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&bar->b1_full[st], C::B_BYTES);
            load_tile(d1, KV ? &tm_q : cmap ? &tm_kc : &tm_k, &bar->b1_full[st], BN, row, h, it.b);
          }
          __syncwarp();
          if (!wait(&bar->b2_empty[st], ph ^ 1u)) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&bar->b2_full[st], C::B_BYTES);
            load_tile(d1 + C::B_BYTES, KV ? &tm_do : cmap ? &tm_vc : &tm_v, &bar->b2_full[st], BN, row, h, it.b);
          }
          __syncwarp();
          ++t;
          if (KV && t == it.nt0) { t = 0; ++g; }
          if (!KV && t == it.nt0 + it.nt1) t = 0;  // (after the walk for delta)
          if (i + 1 == max(n - 1, 1)) prefetch();
        }
        if (failed) break;
      } else {
        prefetch();
      }
      it = nx;
    }
  } else if (KV && warp == C::EXT_WARP) {
    // ------------------------------------------------------------ extra columns
    // Loaded one tile ahead: the stage is waited for with the values in hand.
    const uint4 none = ext_columns<BF16>(p.none, 0.f);
    uint32_t fill = 0;
    for (uint32_t ring = 0;; ++ring) {
      const BwdItem* slot = take_item(ring, tmo);
      if (!slot) break;
      const int nt0 = slot->nt0, n = slot->heads * nt0, row0 = slot->row0, end0 = slot->end0, stat_h = slot->stat_h;
      const uint4* src = p.xstats + slot->stat0;
      // float16, one tile: its columns hold the codes that ds_mul is found from
      const bool one = !BF16 && n == 1 && !streams_several(p, *slot);
      const int v = one ? kv_item_value_code(p, *slot) : 0;
      if (!one) release_item(ring);
      uint4 x[BN / 32];
      int t = 0;
      auto load = [&]() {  // tile t of the head at src, and on to the next
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          const int r = row0 + t * BN + c * 32 + lane;
          x[c] = r < end0 ? __ldg(src + r) : none;
        }
        if (++t == nt0) {
          t = 0;
          src += stat_h;
        }
      };
      if (n > 0) load();
      for (int i = 0; i < n; ++i, ++fill) {
        const int st = fill % STAGES;
        if (!wait(&bar->b1_empty[st], ((fill / STAGES) & 1u) ^ 1u)) break;
        uint8_t* x1 = sBx + st * 2 * C::BX_BYTES;
        bool saturated = false;
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          if (!BF16) saturated |= ext_saturated(x[c]);
          *reinterpret_cast<uint4*>(ext_row(x1, c * 32 + lane, 0)) = make_uint4(x[c].x, x[c].y, 0, 0);
          *reinterpret_cast<uint4*>(ext_row(x1 + C::BX_BYTES, c * 32 + lane, 0)) = make_uint4(0, 0, x[c].z, x[c].w);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->b1_full[st]);
        if (saturated) atomicExch(p.err, kErrStatistics);
        if (i + 1 < n) load();
      }
      if constexpr (!BF16) {
        if (one && !failed) {
          int g = 0, d = 0;
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) {
            float d0, d1, d2, o;
            unf2(unpack2<BF16>(x[c].z), d0, d1);
            unf2(unpack2<BF16>(x[c].w & 0xffffu), d2, o);
            g = max(g, (int)(x[c].w >> 16));
            d = max(d, mag_code(fabsf(fmaf(d0, 0x1p12f, fmaf(d2, 0x1p-12f, d1)))));
          }
          d = __reduce_max_sync(0xffffffffu, d);
          const int power = ds_power(__reduce_max_sync(0xffffffffu, g), v, d);
          if (lane == 0) {
            ring_items[ring & 3].ds_mul = BwdScale<BF16>::kInv * pow2(power);
            mbar_arrive(&bar->mul_full[ring & 3]);
          }
          release_item(ring);
        }
      }
      if (failed) break;
    }
  } else if (KV && warp == C::POWER_WARP) {
    // ------------------------------------------------------------ float16: ds_mul of items of several tiles
    // (A warp for it, since its loads take as long as a short item: moved out of
    // the warp above, 64 packed sequences with contexts 627 -> 608 us.  It waits
    // as long as the item before lasts; what hangs gives up in another warp.)
    if constexpr (KV && !BF16) {
      for (uint32_t ring = 0;; ++ring) {
        const BwdItem* slot = take_item(ring, 1024 * tmo);
        if (!slot) break;
        const bool several = streams_several(p, *slot);
        if (slot->heads * slot->nt0 != 1 || several) {
          const float m = BwdScale<BF16>::kInv * pow2(slot->nt0 > 0 ? kv_item_power(p, *slot, several, lane) : 0);
          if (lane == 0) {
            ring_items[ring & 3].ds_mul = m;
            mbar_arrive(&bar->mul_full[ring & 3]);
          }
        }
        release_item(ring);
      }
    }
  } else if (warp == C::MMA_WARP) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t fmt = BF16 ? 1u : 0u;
    constexpr uint32_t idesc_s = make_idesc_f16(fmt, 0, 0, C::BM, BN);
    constexpr uint32_t idesc_acc = make_idesc_f16(fmt, 0, 1, C::BM, C::DV);
    constexpr uint32_t layout = swizzle_code(SWB);
    const uint32_t a1 = smem_u32(sA), a2 = a1 + C::A_BYTES, sB0 = smem_u32(sB);
    const uint32_t ax = (smem_u32(sAx) >> 4) | (1u << 16), bx0 = (smem_u32(sBx) >> 4) | (1u << 16);
    constexpr uint32_t hi_x = (256u >> 4) | (1u << 14) | (swizzle_code(32) << 29);  // 32-byte rows
    const bool leader = elect_one();
    // high descriptor word: 8-row stride, descriptor version 1, swizzle
    constexpr uint32_t hi = (8 * SWB >> 4) | (1u << 14) | (layout << 29);
    constexpr uint32_t lbo_k = 1u << 16;                // K-major: unused
    constexpr uint32_t lbo_mn = (BN * SWB >> 4) << 16;  // MN-major: slab stride
    // scores: D[128, BN] = A[128, D] B[BN, D]^T (A in TMEM or shared memory;
    // KV: and the extra columns bx), then commit to `done`
    auto issue_scores = [&](uint32_t d, uint32_t a_tm, uint32_t a_base, uint32_t b_base, uint32_t bx, uint64_t* done) {
      if (leader) {
        const uint32_t a = (a_base >> 4) | lbo_k, b = (b_base >> 4) | lbo_k;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t slab = (kk * 32) / SWB, inrow = (kk * 32) % SWB;
          const uint32_t bk = b + ((slab * (BN * SWB) + inrow) >> 4);
          if constexpr (C::ATM) mma_ts(d, a_tm + kk * 8, bk, hi, idesc_s, kk > 0 ? 1u : 0u);
          else mma_ss(d, a + ((slab * (C::BM * SWB) + inrow) >> 4), bk, hi, idesc_s, kk > 0 ? 1u : 0u);
        }
        if constexpr (KV) mma_ss(d, ax, bx, hi_x, idesc_s, 1u);
        umma_commit(done);
      }
    };
    // accumulators: D[128, DV] += A[128, BN] (16-bit, TMEM) B[BN, DV], as A's
    // columns are handed over.  They are in EW_GROUPS pieces, `piece` TMEM
    // columns apart; a half is every other K step.  `rest` (0: none): A's second
    // part, in pieces NC columns apart.
    auto issue_acc = [&](uint64_t* full, uint32_t ph, uint32_t d, uint32_t a_tm, uint32_t piece, uint32_t rest,
                         uint32_t b_base, bool acc, uint64_t* done) -> bool {
      constexpr int KP = C::NC / 16;  // K steps per piece
      constexpr int STEP = C::SPLIT ? KP : 1;
      const uint32_t b = (b_base >> 4) | lbo_mn;
#pragma unroll
      for (int half = 0; half < STEP; ++half) {
        if (!wait(full + half, ph)) return false;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int kk = half; kk < BN / 16; kk += STEP)
            mma_ts(d, a_tm + (kk / KP) * piece + (kk % KP) * 8, b + (kk * 16 * SWB >> 4), hi, idesc_acc,
                   kk > 0 ? 1u : acc ? 1u : 0u);
          if (half == STEP - 1) {
            if (rest != 0) {
#pragma unroll 1
              for (int kk = 0; kk < BN / 16; ++kk)
                mma_ts(d, rest + (kk / KP) * C::NC + (kk % KP) * 8, b + (kk * 16 * SWB >> 4), hi, idesc_acc, 1u);
            }
            umma_commit(done);
          }
        }
      }
      return true;
    };
    auto commit = [&](uint64_t* b) {
      if (leader) umma_commit(b);
    };
    // Rows past the range hold another sequence's rows or padding, NaN perhaps:
    // P and dS are 0 there, but 0 * NaN is not.
    auto clear_rows = [&](uint8_t* tile, int valid) {
      if (valid < BN) {
        for (int s = 0; s < C::NSLAB; ++s) {
          uint4* z = reinterpret_cast<uint4*>(tile + s * (BN * SWB) + valid * SWB);
          for (int i = lane; i < (BN - valid) * SWB / 16; i += 32) z[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
    };
    // Everything below is kept incremental (stage, phase, tiles left in the
    // range): between two MMA batches this warp's own instructions are on the
    // critical path.
    struct Stage {
      uint32_t i = 0, ph = 0;
      __device__ __forceinline__ void next() {
        if (++i == (uint32_t)STAGES) {
          i = 0;
          ph ^= 1u;
        }
      }
    };
    Stage s_st, d_st, c_st;  // stages of the next S, the next dP, the current accumulations
    uint32_t aload = 0, ph = 0, ph2 = 0, acc_ph = 1;  // ph2: of a barrier that every other tile uses (DB)
    for (uint32_t ring = 0;; ++ring) {
      const BwdItem* slot = take_item(ring, tmo);
      if (!slot) break;
      const int nt0 = slot->nt0, nt1 = slot->nt1, pre = KV ? 0 : slot->pre, n = slot->heads * nt0 + nt1 + pre;
      // valid rows of each range's last tile
      const int last0 = slot->end0 - slot->row0 - (nt0 - 1) * BN, last1 = slot->end1 - slot->row1 - (nt1 - 1) * BN;
      const uint32_t dh_off = (slot->dh * C::DV / C::SLAB_COLS) * (BN * SWB);
      const bool few = slot->few != 0;
      const uint32_t rest_p = few ? tmem_base + C::TM_S + C::NC / 2 : 0;
      release_item(ring);
      if (n == 0) continue;
      if (!wait(C::ATM ? &bar->a_tm : &bar->a_full, aload & 1u)) break;
      ++aload;
      // Tiles left in the range that S / dP walk (KV: its one range, once per
      // head; Q: one range, or the two in turn), and that range's last tile.
      int s_left = nt0 > 0 ? nt0 : nt1, d_left = s_left;
      int s_last = nt0 > 0 ? last0 : last1, d_last = s_last;
      bool s_second = nt0 == 0, d_second = s_second;
      auto next_range = [&](bool& second, int& left, int& last) {
        if (!KV) second = second ? nt0 == 0 : nt1 > 0;
        left = second ? nt1 : nt0;
        last = second ? last1 : last0;
      };
      auto do_s = [&]() -> bool {
        if (!wait(&bar->b1_full[s_st.i], s_st.ph)) return false;
        if (--s_left == 0) {
          if (s_last < BN) clear_rows(sB + s_st.i * 2 * C::B_BYTES, s_last);
          next_range(s_second, s_left, s_last);
        }
        tc_fence_after();
        issue_scores(tmem_base + C::TM_S, tmem_base + C::TM_A1, a1, sB0 + s_st.i * 2 * C::B_BYTES,
                     bx0 + s_st.i * (2 * C::BX_BYTES >> 4), &bar->s_full);
        s_st.next();
        return true;
      };
      auto do_dp = [&](uint32_t db) -> bool {  // into buffer db
        if (!wait(&bar->b2_full[d_st.i], d_st.ph)) return false;
        if (--d_left == 0) {
          if (d_last < BN) clear_rows(sB + d_st.i * 2 * C::B_BYTES + C::B_BYTES, d_last);
          next_range(d_second, d_left, d_last);
        }
        tc_fence_after();
        issue_scores(tmem_base + C::TM_DP + (C::DB ? db * BN : 0u), tmem_base + C::TM_A2, a2, sB0 + d_st.i * 2 * C::B_BYTES + C::B_BYTES,
                     bx0 + ((d_st.i * 2 + 1) * C::BX_BYTES >> 4), &bar->dp_full[C::DB ? db : 0u]);
        if (!KV) commit(&bar->b2_empty[d_st.i]);
        d_st.next();
        return true;
      };
      if (!do_s() || !do_dp(ph)) break;
      bool ok = true;
      for (int left = n; left > 0; --left, ph2 ^= ph, ph ^= 1u) {
        const uint32_t db = C::DB ? ph : 0u, ds_ph = C::DB ? ph2 : ph;
        const uint32_t t_ds = tmem_base + C::TM_DP + db * BN;
        const bool more = left > 1, first = left == n - pre;  // (first to accumulate)
        const uint32_t b1 = sB0 + c_st.i * 2 * C::B_BYTES + dh_off, b2 = b1 + C::B_BYTES;
        if (!C::ATM && !more) commit(&bar->a_empty);  // every S and dP of the item is issued
        // The next S as soon as its columns are free: this S is in registers,
        // and (KV, P over S) P is consumed, the MMAs running in order.  One
        // stage only: its tile B1 takes the place of the one dS still needs.
        // P's second part is over S (a separate P's too), so that S waits as well.
        constexpr bool kEarlyS = C::SEP_P || !KV;
        const bool early = kEarlyS && !(KV && few);
        if (kEarlyS && STAGES > 1) {
          if (!wait(&bar->s_free, ph) || (early && more && !do_s())) { ok = false; break; }
          // (The other buffer's dS was read by the accumulation issued last.)
          if (C::DB && more && !do_dp(ph ^ 1u)) { ok = false; break; }
        }
        if (first) {
          if (!wait(&bar->acc_empty, acc_ph)) { ok = false; break; }
          acc_ph ^= 1u;
        }
        if constexpr (KV) {
          if (!issue_acc(bar->p_full, ph, tmem_base + C::TM_ACC1, tmem_base + C::TM_P, C::SEP_P ? C::NC / 2 : C::NC,
                         rest_p, b2, !first, &bar->b2_empty[c_st.i])) { ok = false; break; }
          if (C::SEP_P) commit(&bar->p_free);
        }
        if (!early && STAGES > 1 && more && !do_s()) { ok = false; break; }
        if (!KV && left > n - pre) {  // delta only: dP is read, B1 is free
          if (!wait(&bar->ds_full[db], ds_ph)) { ok = false; break; }
          commit(&bar->b1_empty[c_st.i]);
        } else if (!issue_acc(&bar->ds_full[db], ds_ph, tmem_base + C::TM_ACC2, t_ds, C::NC,
                              few ? t_ds + C::NC / 2 : 0, b1, !first, &bar->b1_empty[c_st.i])) {
          ok = false;
          break;
        }
        c_st.next();
        if (more) {
          if ((STAGES == 1 && !do_s()) || (!C::DB && !do_dp(ph ^ 1u))) { ok = false; break; }
        } else {
          commit(&bar->acc_full);
        }
      }
      if (!ok) break;
    }
  } else {
    // ------------------------------------------------------------ element-wise warps + epilogue
    const int g = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    constexpr int NC = C::NC;
    const uint32_t tS = tmem_base + lane_off + C::TM_S + g * NC;
    const uint32_t tDP0 = tmem_base + lane_off + C::TM_DP + g * NC;
    const uint32_t tP = C::SEP_P ? tmem_base + lane_off + C::TM_P + g * (NC / 2) : tS;
    constexpr float kInv = BwdScale<BF16>::kInv;
    const F2 sl2_2 = f2(p.scale_log2, p.scale_log2);
    uint32_t ph = 0, ph2 = 0, acc_ph = 0, aload = 0, sums = 0;  // ph2: of a barrier that every other tile uses (DB)
    auto next_tile = [&]() {
      ph2 ^= ph;
      ph ^= 1u;
    };
    auto arrive = [&](uint64_t* b) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    auto ld = [&](uint32_t a, uint32_t(&r)[NC]) {
      if constexpr (NC == 32) tmem_ld_x32(a, r); else tmem_ld_x16(a, r);
    };
    // Stores packed pairs, half h of them with SPLIT; give hands them over.
    auto put = [&](uint32_t a, const uint32_t(&r)[NC / 2], int h) {
      if constexpr (C::SPLIT) tmem_st_x8_nowait(a + h * 8, r + h * 8);
      else if constexpr (NC == 32) tmem_st_x16_nowait(a, r);
      else tmem_st_x8_nowait(a, r);
    };
    auto give = [&](uint32_t a, const uint32_t(&r)[NC / 2], int h, uint64_t* full) {
      put(a, r, h);
      tmem_wait_st();
      arrive(full + h);
    };
    constexpr int HALVES = C::SPLIT ? 2 : 1, HC = NC / 2 / HALVES;  // pairs per half
    // Stationary tiles, shared memory -> TMEM: half the warps copy A1, half A2,
    // (D > 16) each warp half of its rows' columns.
    auto copy_a = [&]() -> bool {
      if (!wait(&bar->a_full, aload & 1u)) return false;
      ++aload;
      constexpr int W = D > 16 ? D / 4 : 8;  // 32-bit words per thread
      const int half = D > 16 ? g & 1 : 0;
      if (D > 16 || (g & 1) == 0) {
        const uint8_t* tile = sA + (g >> 1) * C::A_BYTES;
        uint32_t v[W];
#pragma unroll
        for (int c = 0; c < W / 4; ++c) {
          const uint4 x = ld_swizzled<SWB>(tile, C::BM, row, half * (W / 4) + c);
          v[4 * c] = x.x; v[4 * c + 1] = x.y; v[4 * c + 2] = x.z; v[4 * c + 3] = x.w;
        }
        const uint32_t dst = tmem_base + lane_off + ((g >> 1) ? C::TM_A2 : C::TM_A1) + half * W;
        if constexpr (W == 64) tmem_st_x64(dst, v);
        else if constexpr (W == 32) tmem_st_x32(dst, v);
        else if constexpr (W == 16) tmem_st_x16(dst, v);
        else tmem_st_x8(dst, v);
      }
      arrive(&bar->a_tm);
      if (lane == 0) mbar_arrive(&bar->a_empty);
      return true;
    };
    // Results wait in registers (16-bit pairs) until the next item's first
    // scores are in hand: their stores then drain behind its exponentials
    // instead of in front of them (up to 32 columns; 64, in 32 registers, lost
    // at D = 128: KV pass 123 -> 131 us).  KV: groups 0, 1 hold halves of dV, groups
    // 2, 3 halves of dK; Q: quarters of dQ.
    constexpr int PARTS = KV ? 2 : 4;
    constexpr int COLS = C::DV / PARTS >= 16 ? C::DV / PARTS : 16;
    constexpr bool kDefer = COLS <= 32;
    const int part = KV ? g & 1 : g;
    const bool is_dv = KV && g < 2;
    uint32_t res[COLS / 2];
    T* res_dst = nullptr;
    auto flush = [&]() {
      if (res_dst != nullptr) {
#pragma unroll
        for (int c = 0; c < COLS / 16; ++c) st_sector(res_dst + c * 16, res + 8 * c);
      }
      res_dst = nullptr;
    };
    const BwdItem* it = take_item(0, tmo);
    if (C::ATM && it && it->heads * it->nt0 + it->nt1 > 0 && !copy_a()) it = nullptr;
    for (uint32_t ring = 0; it; ++ring) {
      const int nt0 = it->nt0, pre = KV ? 0 : it->pre, n = it->heads * nt0 + it->nt1 + pre;
      float2 rs = make_float2(0.f, 0.f);
      if (!KV && row < it->valid) rs = __ldg(p.stats + it->out_row + row);
      // What takes P (dP - delta) to the dS that is held (KV, float16: it->ds_mul).
      float ds_mul = kInv;
      if constexpr (!KV && !BF16) {
        const int code = row < it->valid ? reinterpret_cast<const unsigned short*>(p.xstats + it->out_row + row)[7] : 0;
        if (n > 0) ds_mul *= pow2(ds_power(code, q_item_value_code(p, *it, lane), mag_code(fabsf(rs.y))));
      }
      const F2 mul_2 = f2(ds_mul, ds_mul);
      const F2 nl_2 = f2(rs.x, rs.x);
      F2 nd_2 = f2(rs.y * ds_mul, rs.y * ds_mul);
      // (The first tile apart, so that the waiting results leave their registers
      // there; and apart the items of few terms, of which some sum delta themselves.)
      auto tile = [&](auto first, auto few, int i) -> bool {
        constexpr bool kFew = decltype(few)::value;
        const uint32_t db = C::DB ? ph : 0u, tDP = tDP0 + db * BN;
        if (!wait(&bar->s_full, ph)) return false;
        tc_fence_after();
        uint32_t x[NC];
        F2 pr[NC / 2];
        ld(tS, x);
        if (C::SEP_P || !KV) arrive(&bar->s_free);
        if constexpr (kDefer && decltype(first)::value) flush();
        uint32_t pk[NC / 2], pk2[NC / 2];  // (pk2: few only)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
#pragma unroll
          for (int c = h * HC; c < (h + 1) * HC; ++c) {
            const F2 xs = f2u(x[2 * c], x[2 * c + 1]);
            float a, b;
            unf2(KV ? mul2(xs, sl2_2) : fma2(xs, sl2_2, nl_2), a, b);
            pr[c] = f2(ex2_approx(a), ex2_approx(b));
          }
          if constexpr (KV) {
#pragma unroll
            for (int c = h * HC; c < (h + 1) * HC; ++c) {
              pk[c] = pack2<BF16>(pr[c]);
              if constexpr (kFew) pk2[c] = pack_rest<BF16>(pr[c], pk[c]);
            }
            if (C::SEP_P) {
              if (!wait(&bar->p_free, ph ^ 1u)) return false;
              tc_fence_after();
            }
            if constexpr (kFew) put(tS + NC / 2, pk2, h);
            give(tP, pk, h, bar->p_full);
          }
        }
        if constexpr (KV && !BF16) {  // (here, with few registers in use; at dS, where it spills: 608 -> 617 us)
          if (i == 0 && !wait(&bar->mul_full[ring & 3], (ring >> 2) & 1u)) return false;
          const float m = it->ds_mul;
#pragma unroll
          for (int c = 0; c < NC / 2; ++c) pr[c] = mul2(pr[c], f2(m, m));
        }
        if constexpr (!KV) {
          const int j = kFew && i >= pre ? i - pre : i;
          const int valid = (j >= nt0 ? it->end1 - (it->row1 + (j - nt0) * BN) : it->end0 - (it->row0 + j * BN)) - g * NC;
          if (valid < NC) {
#pragma unroll
            for (int c = 0; c < NC / 2; ++c) {
              float a, b;
              unf2(pr[c], a, b);
              pr[c] = f2(2 * c < valid ? a : 0.f, 2 * c + 1 < valid ? b : 0.f);
            }
          }
        }
        if (!wait(&bar->dp_full[db], C::DB ? ph2 : ph)) return false;
        tc_fence_after();
        ld(tDP, x);
        if constexpr (!KV && kFew) {
          if (i < pre || n == 1) {
            F2 acc = f2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < NC / 2; ++c) acc = fma2(pr[c], f2u(x[2 * c], x[2 * c + 1]), acc);
            float a, b;
            unf2(acc, a, b);
            float* part = sSum + (sums & 1u) * (C::EW_GROUPS * C::BM) + row;
            part[g * C::BM] = i == 0 ? a + b : part[g * C::BM] + (a + b);
            if (i == pre - 1 || n == 1) {
              // The four column groups' parts, in the same order by all.
              __syncwarp();
              if (lane == 0) mbar_arrive(&bar->sum_full);
              if (!wait(&bar->sum_full, sums & 1u)) return false;
              ++sums;
              const float nd = -((part[0] + part[C::BM]) + (part[2 * C::BM] + part[3 * C::BM])) * kInv;
              nd_2 = f2(nd * ds_mul, nd * ds_mul);
              if (g == 0) {
                if (row < it->valid) {
                  const uint4 e = ext_columns<BF16>(0.f, nd);
                  uint4* dst = p.xstats + it->out_row + row;
                  dst->z = e.z;
                  reinterpret_cast<unsigned short*>(dst)[6] = (unsigned short)e.w;
                }
                if constexpr (!BF16) {
                  const int d = __reduce_max_sync(0xffffffffu, row < it->valid ? mag_code(fabsf(nd)) : 0);
                  if (lane == 0) atomicMax(&p.range[it->out_row].y, d);
                }
              }
            }
            if (i < pre) {
              arrive(&bar->ds_full[db]);
              next_tile();
              return true;
            }
          }
        }
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
#pragma unroll
          for (int c = h * HC; c < (h + 1) * HC; ++c) {
            F2 d = f2u(x[2 * c], x[2 * c + 1]);
            if constexpr (!KV) d = fma2(d, mul_2, nd_2);
            d = mul2(pr[c], d);
            pk[c] = pack2<BF16>(d);
            if constexpr (kFew) pk2[c] = pack_rest<BF16>(d, pk[c]);
          }
          if constexpr (kFew) put(tDP + NC / 2, pk2, h);
          give(tDP, pk, h, &bar->ds_full[db]);
        }
        next_tile();
        return true;
      };
      using Yes = std::true_type;
      using No = std::false_type;
      if (n > 0 && it->few) {
        flush();
        for (int i = 0; i < n && tile(No(), Yes(), i); ++i) {}
      } else if (n > 0 && tile(Yes(), No(), 0)) {
        for (int i = 1; i < n && tile(No(), No(), i); ++i) {}
      }
      if (failed) break;
      // dP of the last tile was the last MMA to read the stationary tiles (and
      // came after the last S), so the next item's can move in: its first
      // scores follow this item's last accumulations at once.
      const BwdItem* next = take_item(ring + 1, tmo);
      if (failed) break;
      const int next_n = next ? next->heads * next->nt0 + next->nt1 : 0;
      if (C::ATM && next_n > 0 && !copy_a()) break;
      const int valid = it->valid, limit = it->limit;
      if (part * COLS < C::DV && row < limit && (KV || p.dq != nullptr)) {
        T* base = reinterpret_cast<T*>(!KV ? p.dq : is_dv ? (it->a_map ? p.dvc : p.dv) : (it->a_map ? p.dkc : p.dk));
        res_dst = base + (it->out_row + row) * (long long)D + it->dh * C::DV + part * COLS;
      }
      if (n > 0) {
        if (!wait(&bar->acc_full, acc_ph)) break;
        acc_ph ^= 1u;
        tc_fence_after();
        if (part * COLS < C::DV) {
          const uint32_t tO = tmem_base + lane_off + (is_dv ? C::TM_ACC1 : C::TM_ACC2) + part * COLS;
          const float fs = is_dv ? kInv : BF16 ? p.scale : p.scale * kInv * inv_pow2(KV ? it->ds_mul : ds_mul);
          const F2 f = f2(fs, fs);
#pragma unroll
          for (int c0 = 0; c0 < COLS; c0 += 16) {
            uint32_t o[16];
            tmem_ld_x16(tO + c0, o);
            const int at = kDefer ? c0 / 2 : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) res[at + e] = row < valid ? pack2<BF16>(mul2(f2u(o[2 * e], o[2 * e + 1]), f)) : 0u;
            if (!kDefer && res_dst != nullptr) st_sector(res_dst + c0, res);
          }
        }
        if (!kDefer) res_dst = nullptr;
        arrive(&bar->acc_empty);
      } else {
#pragma unroll
        for (int e = 0; e < COLS / 2; ++e) res[e] = 0u;
      }
      if (next_n == 0 || !kDefer) flush();
      release_item(ring);
      it = next;
    }
  }

  // ------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::MMA_WARP) {
    if (*abort_flag) {
      // Give in-flight MMAs a bounded chance to retire before freeing TMEM.
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 1000000ull) {}
    }
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

struct BwdRows {  // v, or the context's: [batch][heads][rows][D] in strides of elements
  const uint16_t* data;
  long long batch, head, row;
};

// Sum over the LANES neighbouring threads that share a row.
template <int LANES>
__device__ __forceinline__ float row_sum(float s) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// a . b over a vector of eight 16-bit numbers
template <bool BF16>
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b) {
  const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x0, x1, y0, y1;
    unf2(unpack2<BF16>(av[e]), x0, x1);
    unf2(unpack2<BF16>(bv[e]), y0, y1);
    s = fmaf(x0, y0, fmaf(x1, y1, s));
  }
  return s;
}

// The code of the largest norm among `rows` rows (at most 128) from src on, over
// the lanes of a warp, by THREADS threads of which this is number t.
template <int D, int THREADS>
__device__ __forceinline__ int largest_norm_code(const uint16_t* src, long long stride, int rows, int t) {
  constexpr int LANES = D / 8, STEP = THREADS / LANES;
  src += (t % LANES) * 8;
  float m = 0.f;
#pragma unroll 8
  for (int r0 = 0; r0 < rows; r0 += STEP) {
    const int r = r0 + t / LANES;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r < rows) x = __ldg(reinterpret_cast<const uint4*>(src + r * stride));
    m = fmaxf(m, row_sum<LANES>(dot8<false>(x, x)));
  }
  return __reduce_max_sync(0xffffffffu, mag_code_of_square(m));
}

// Per output row: {-lse * log2(e) + kPExp, -rowsum(dO * O)}, in float32 and as
// the KV pass's extra columns; also zeroes the item counters of the two passes
// that follow.  Reads O and dO once (bound by HBM).  delta uses the 16-bit O that
// the forward pass returned (what that costs: at the head of this file).
// float16: also the rows' codes of |dO| and each tile's largest; the blocks behind
// do the same for v's tiles.  A block takes SLOTS tile slots of 128 rows: one, or
// eight (a warp each) where there are many of few rows (4096 sequences of 1 to 16
// tokens, 8 heads: 26 us, one slot a block 103; 16 sequences of 512, 32 heads of
// 128: one slot a block 27 us, eight 52).
template <int D, bool BF16, int SLOTS>
__global__ void __launch_bounds__(256) attn_bwd_stats_kernel(const BwdParams p, const uint4* __restrict__ out,
                                                             const uint4* __restrict__ dout,
                                                             const float* __restrict__ lse, float ext_mul, const BwdRows v) {
  constexpr int THREADS = 256 / SLOTS, LANES = D / 8, STEP = THREADS / LANES;
  __shared__ int code[2];  // (one slot: its largest)
  const int lane = threadIdx.x & 31, tid = threadIdx.x % THREADS;
  if (blockIdx.x == 0 && threadIdx.x < 2) p.counter[threadIdx.x] = 0;
  if constexpr (!BF16 && SLOTS == 1) {
    if (threadIdx.x < 2) code[threadIdx.x] = 0;
    __syncthreads();
  }
  long long i = (long long)blockIdx.x * SLOTS + threadIdx.x / THREADS;
  const long long nq = (long long)p.H * p.slots;
  const bool is_v = i >= nq;
  if (is_v) i -= nq;
  if (is_v && (BF16 || i >= (long long)p.HK * p.slots)) return;
  const int heads = is_v ? p.HK : p.H, h = (int)i / p.slots, slot = (int)i - h * p.slots;
  int b = 0, r0, rows;  // batch coordinate, first row, rows from there on
  long long first;      // the first row in the order of the output (or of k)
  if (p.layout == FMLM_BWD_PACKED) {
    const int s = find_slot_owner(p.cu_q, p.B, slot, lane);
    int s0, s1;
    packed_rows(p, s, s0, s1);
    const int t = slot - ((s0 >> 7) + s);
    r0 = s0 + t * 128;
    rows = t >= 0 ? s1 - r0 : 0;
    first = (long long)h * p.T + r0;
  } else {
    const int per_seq = (p.N + 127) / 128;
    b = slot / per_seq;
    r0 = (slot % per_seq) * 128;
    int L = p.N;
    if (p.layout == FMLM_BWD_PADDED) L = min(max(__ldg(p.cu_q + b + 1) - __ldg(p.cu_q + b), 0), p.N);
    rows = L - r0;
    first = ((long long)b * heads + h) * p.N + r0;
  }
  rows = min(rows, 128);
  if (rows <= 0) return;
  // the largest over the slot's threads, valid in its thread 0
  auto largest = [&](int c, int* shared) {
    if constexpr (SLOTS == 1) {
      if (lane == 0) atomicMax(shared, c);
      __syncthreads();
      return *shared;
    } else {
      return c;
    }
  };
  if constexpr (!BF16) {
    if (is_v) {
      const int c = largest(largest_norm_code<D, THREADS>(v.data + b * v.batch + h * v.head + r0 * v.row, v.row, rows, tid), code);
      if (tid == 0) *reinterpret_cast<int2*>(&p.range[first].z) = make_int2(c, 0);
      return;
    }
  }
  int g_max = 0, d_max = 0;
  const uint4 *o = out + first * LANES + tid, *d = dout + first * LANES + tid;
  float2* stats = const_cast<float2*>(p.stats);
#pragma unroll 4
  for (int rb = 0; rb < rows; rb += STEP, o += THREADS, d += THREADS) {
    const int r = rb + tid / LANES;
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    float l = 0.f;
    if (r < rows) {
      x = __ldg(o);
      y = __ldg(d);
      l = __ldg(lse + first + r);
    }
    const float s = row_sum<LANES>(dot8<BF16>(x, y));
    float g = 0.f;
    if constexpr (!BF16) g = row_sum<LANES>(dot8<BF16>(y, y));
    if (r < rows && tid % LANES == 0) {
      const float nl = fmaf(-1.4426950408889634f, l, BwdScale<BF16>::kPExp);
      stats[first + r] = make_float2(nl, -s);
      uint4 e = ext_columns<BF16>(nl * ext_mul, -s);
      if constexpr (!BF16) {
        const int c = mag_code_of_square(g);
        e.w |= (uint32_t)c << 16;
        g_max = max(g_max, c);
        d_max = max(d_max, mag_code(fabsf(s)));
      }
      p.xstats[first + r] = e;
    }
  }
  if constexpr (!BF16) {
    g_max = largest(__reduce_max_sync(0xffffffffu, g_max), &code[0]);
    d_max = largest(__reduce_max_sync(0xffffffffu, d_max), &code[1]);
    if (tid == 0) *reinterpret_cast<int2*>(&p.range[first].x) = make_int2(g_max, d_max);
  }
}

// float16, packed: what range_by_sequence needs.  The first blocks find the code
// of the largest |v| of each context, SLOTS slots of 128 rows each, and leave it at
// the sequence that sees it (a shared context's at the head's first row; the
// kernel before zeroed it).  The others gather the tiles' codes of a sequence and
// head, a warp each; for v also those of the sequences before it.  Maxima of whole
// numbers do not depend on their order.
template <int D, int SLOTS>
__global__ void __launch_bounds__(128) attn_bwd_range_kernel(const BwdParams p, const BwdRows vc, int context_blocks) {
  const int lane = threadIdx.x & 31;
  if ((int)blockIdx.x < context_blocks) {
    constexpr int THREADS = 128 / SLOTS;
    const long long i = (long long)blockIdx.x * SLOTS + threadIdx.x / THREADS;
    const int h = (int)(i / p.cslots), slot = (int)(i % p.cslots);
    if (h >= p.HK) return;
    const int c = find_slot_owner(p.cu_c, p.C, slot, lane);
    const int c0 = min(max(__ldg(p.cu_c + c), 0), p.Tc), c1 = min(max(__ldg(p.cu_c + c + 1), 0), p.Tc);
    const int t = slot - ((c0 >> 7) + c), r0 = c0 + t * 128, rows = t >= 0 ? min(c1 - r0, 128) : 0;
    int q0 = 0, q1 = 1;
    if (p.C > 1) packed_rows(p, c, q0, q1);
    if (rows <= 0 || q1 <= q0) return;  // (an entry that no query sees)
    const int x = largest_norm_code<D, THREADS>(vc.data + h * vc.head + r0 * vc.row, vc.row, rows, threadIdx.x % THREADS);
    if (lane == 0) atomicMax(&p.range[(long long)h * p.T + q0].w, x);
    return;
  }
  const long long i = (long long)(blockIdx.x - context_blocks) * 4 + (threadIdx.x >> 5);  // query heads, then v's
  const int head = (int)(i / p.B), b = (int)(i % p.B);
  if (head >= p.H + p.HK) return;
  const bool is_v = head >= p.H;
  int4* x = p.range + (long long)(is_v ? head - p.H : head) * p.T;
  int s0, s1;
  packed_rows(p, b, s0, s1);
  if (s1 <= s0) return;
  int g = 0, d = 0;  // (v: its code in g, that of all sequences up to it in d)
  for (int r = s0 + lane * 128; r < s1; r += 32 * 128) {
    g = max(g, (is_v ? x[r].z : x[r].x) & 255);  // (z may have been gathered already)
    if (!is_v) d = max(d, x[r].y);
  }
  g = __reduce_max_sync(0xffffffffu, g);
  if (is_v && p.causal) {
    d = g;
    for (int e = lane; e < b; e += 32) {
      int e0, e1;
      packed_rows(p, e, e0, e1);
      for (int r = e0; r < e1; r += 128) d = max(d, x[r].z & 255);
    }
  }
  d = __reduce_max_sync(0xffffffffu, d);
  if (lane != 0) return;
  if (is_v) x[s0].z = g | d << 8;
  else *reinterpret_cast<int2*>(x + s0) = make_int2(g, d);
}

}  // namespace fmlm
