// Attention of a chunk of new tokens over the paged cache alone, on the 5th-generation tensor cores.
//
// The keys and values of the new tokens have been appended to the pages before the call (by fill_kv_pages or
// fill_kv_pages_rotary), so queries attend to pages only: with sequence s of length L bringing n query rows, row i stands at
// position L - n + i and sees the keys [max(0, position - window + 1), position] (causal), or all L keys.  One kernel serves
// single tokens, proposed tokens to verify and prompt chunks, in any mix.
//
// Rows.  The query heads of one kv head are packed into the rows of an accumulator tile, token by token: with G heads per kv
// head a tile of M = 128 rows holds 128 / G tokens (rows past G * (128 / G) are unused).  One TMA box of a 3-D view of the
// queries fetches it.  Short chunks so fill the tile G times better than one head per tile would, and a page is read once
// per kv head and row tile.
//
// Work.  An item is (sequence, kv head, row tile) - up to two accumulator tiles, NQ * 128 / G tokens - and costs its 128-key
// tiles plus a constant.  Every CTA of the persistent grid (one per SM) computes the same prefix sums of these costs over the
// batch and takes an equal share of the line they form; an item that a share's border cuts leaves un-normalised triples
// (m, l, acc) in the workspace, at most two per CTA, which a second small kernel merges.  So one long sequence, many short
// ones and ragged mixes load the SMs equally without the host knowing a length, and the order of every sum is fixed.
//
// Pair and alternate.  An item of more than 128 rows gives each of the two accumulators its own rows; both read the same
// key tiles (pair).  With at most 128 rows both accumulators hold the same rows and take the even and the odd key tiles, so
// that the chain QK^T -> softmax -> PV of one tile overlaps that of the next; they are merged through shared memory at the
// item's end (alternate).
//
//   warp 0      walks the CTA's share, publishes its segments in a ring in shared memory, loads Q and V
//   warp 1      issues the MMAs of S = Q K^T, warp 2 those of O += P V
//   warp 3      loads K
//   warps 4..   one softmax warpgroup per accumulator: thread = row = TMEM lane
//
// Operand layouts are those of the prefill kernel (prefill_tcgen05.cuh): Q K-major with the 128-byte swizzle; a key tile
// copied chunk by chunk from the pages as [D/8][128 tokens][16 B], K-major without swizzle; V pages [D][TPP] K-major with
// the 32- or 64-byte swizzle.
//
// TMEM: a buffer of 128 fp32 scores (two for head_dim <= 64), a P tile of 64 columns per accumulator, the O tiles.  P does not
// overwrite the scores: the softmax warps hold a whole row of them in registers, so the score buffer is free after one read
// and takes the next QK^T, of the other accumulator, while the exponentials are computed.  (With P over S, as the prefill kernel
// has it, softmax, PV and the next QK^T of an accumulator form a chain: 4270 cycles per 2 x 128 x 128 scores at head_dim 128.)
#pragma once

#include <type_traits>

#include "prefill_tcgen05.cuh"

namespace pal {
namespace {

// Costs on the line of items, in quarters of a key tile for two tiles of rows (560 ns of a CTA's time at head_dim 128).  Such a
// tile is bound by the softmax (4 units); for a single one it is bound by the loads of keys and values, 64 KB at head_dim 128 and
// half at 64 (3 and 2).  Tiles with the residual of P hold their score buffer until their PV has run: 512 rows a sequence over
// 8192 keys take 3.4 to 3.8 times as long with it at head_dim 80 to 128 (one score buffer; 14), 2.0 at 32 and 64 (two; 8), 1.6 at 256
// (7); single tiles of rows 2.2 to 2.5 and 1.6 to 1.8 times (7 and 4).  Query load, pipeline fill, masked tiles and output come on
// top: four key tiles' worth for a pair of row tiles, five to six for a single one.  (45 single tokens over 64 to 6000, 16 heads
// of 64: 209 us with two for a single one, CTAs with many short items then end at 187 us and the median at 123; 160-166 us with
// five or six.  The same over 8 heads of 128: 139 and 125.  The constants of the other head sizes follow these two.)
constexpr int kChunkMinShare = 4;  // smallest share of a CTA; it also holds a whole key tile of every kind that occurs
constexpr int kSegRing = 4;

// What one CTA does with one item: key tiles [kt0, kt1) for the rows of the item.
struct ChunkWork {
  int seq, kv_head;
  int head0, heads;    // first query head of the tile, and how many of its heads exist
  int row0, tokens;    // first query row (token) and how many of the item's tokens exist
  int pos0;            // position of the first token (may be negative)
  int kt0, kt1;
  int key_lo, key_hi;  // keys that some row of the item sees
  int key_cap;         // keys of the sequence
  int alternate;       // one tile of rows: the accumulators take even and odd key tiles
  int residual;        // the rounding residual of P takes part
  int slot;            // partial slot to write, -1 = the output itself
  int end;
  // Keys that some rows of the item see and others do not: [some_hi, key_hi) at the diagonal, [key_lo, some_lo) at the start of
  // the windows.  Each range touches at most three key tiles; `bad` marks the keys whose value is not finite.
  int some_lo, some_hi;
  int any_bad;
};
struct ChunkSegment : ChunkWork {
  uint32_t bad[6][4];  // three tiles of the diagonal's range, three of the windows'
};

struct ChunkParams {
  const void* k_pool;
  const void* v_pool;
  const uint32_t* page_table;
  const int32_t* seq_lens;
  const int32_t* cu_seqlens;  // null = every sequence has tokens_per_seq rows
  void* out;
  WaitCtx status;
  int out_f32, causal, window;
  int num_seqs, tokens_per_seq, num_q_heads, num_kv_heads, group;
  int tile_heads, head_blocks, tile_tokens;  // heads and tokens of one accumulator tile, blocks of tile_heads per kv head
  int max_pages_per_seq;
  long long num_pages, total_tokens;
  float scale_log2;
  ChunkCut* cuts;   // [grid]
  float* part_acc;  // [2 * grid][part_rows][D]
  float* part_ml;   // [2 * grid][part_rows][2]: m (log2 units), l
  int part_rows;
};

struct ChunkSeq {
  int row0, n, len, cap;
};

__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int s, int tpp) {
  ChunkSeq q;
  if (p.cu_seqlens) {
    const int total = (int)p.total_tokens;
    const int a = min(max(p.cu_seqlens[s], 0), total), b = min(max(p.cu_seqlens[s + 1], a), total);
    q.row0 = a;
    q.n = b - a;
  } else {
    q.row0 = s * p.tokens_per_seq;
    q.n = p.tokens_per_seq;
  }
  q.len = max(p.seq_lens[s], 0);
  const long long room = p.num_pages > 0 ? (long long)p.max_pages_per_seq * tpp : 0;
  q.cap = (int)min((long long)q.len, room);
  return q;
}

// Keys [lo, hi) that tokens [ta, tb) of the sequence see between them, and their number of 128-key tiles.
__device__ __forceinline__ int chunk_keys(const ChunkParams& p, const ChunkSeq& q, int ta, int tb, int& lo, int& hi) {
  const int base = q.len - q.n;
  hi = p.causal ? min(base + tb, q.cap) : q.cap;
  lo = 0;
  if (p.window > 0 && base + ta >= p.window) lo = base + ta - p.window + 1;
  if (hi <= lo) {
    lo = hi = 0;
    return 0;
  }
  return (hi + kTile - 1) / kTile - lo / kTile;
}

// bf16 rounds P by up to half a step, 2^-8, of its value.  The sum over many keys averages that out; a row of few keys shows it, in
// a bf16 result too: below 256 keys results miss 2e-3 and one unit in the last place (single tokens over 2 to 16 keys, 32 heads of
// 128: one element in 3000).  So an item one of whose rows sees fewer than 256 keys gets the residual P - bf16(P) through a second
// set of PV MMAs, as in the prefill kernel, and every item of a caller who asks for float32.  (For every item of one tile of rows:
// 64 times 4 tokens over 1024 to 4096 take 317 us instead of 156.)  `ta`: the item's first token, which sees the fewest keys.
constexpr int kResidualKeys = 256;
template <typename T>
__device__ __forceinline__ bool chunk_feeds_residual(const ChunkParams& p, const ChunkSeq& q, int ta) {
  if (!Mma16816<T>::kSplitP) return false;
  const int keys = p.causal ? min(q.len - q.n + ta + 1, q.cap) : q.cap;
  return p.out_f32 != 0 || (p.window > 0 ? min(keys, p.window) : keys) < kResidualKeys;
}

// The cost of the item that starts at token `ta` of its sequence: of a key tile, and before the first.
struct ChunkCost {
  int tile, setup;
};
template <typename T, int D, int NQ>
__device__ __forceinline__ ChunkCost chunk_cost(const ChunkParams& p, const ChunkSeq& q, int ta) {
  const bool residual = chunk_feeds_residual<T>(p, q, ta);
  if (NQ == 1) return ChunkCost{residual ? 7 : 4, 16};
  if (q.n - ta > p.tile_tokens) return ChunkCost{residual ? (D <= 64 ? 8 : 14) : 4, 16};
  return D <= 64 ? ChunkCost{residual ? 4 : 2, 12} : ChunkCost{residual ? 7 : 3, 14};
}

template <int D_, int TPP_, int NQ_>
struct ChunkCfg {
  static constexpr int D = D_, TPP = TPP_, NQ = NQ_;
  using Base = TcCfg<D, TPP, NQ, 1>;  // operand tile sizes and ring depth
  // TMEM columns: S buffers (128 fp32 scores), a P tile per accumulator (128 weights, two to a column), O tiles
  static constexpr int kSBuffers = D <= 64 ? 2 : 1;
  static constexpr int kPCol = kSBuffers * kTile;
  static constexpr int kOCol = kPCol + NQ * 64;
  static_assert(kOCol + NQ * Base::DP <= 512, "TMEM holds 512 columns");
  static constexpr int kThreads = 128 + 128 * NQ;
  // K and V ring: two tiles of each (64 KB) in flight, four where they are half as large, one of head_dim 256
  static constexpr int ST = D <= 64 ? 4 : D <= 128 ? 2 : 1;
  static constexpr int kQ = 0;
  static constexpr int kK = NQ * Base::kTileBytes;
  static constexpr int kV = kK + ST * Base::kTileBytes;
  static constexpr int kStage = kV + ST * Base::kTileBytes;  // 4 KB per softmax warp on the way out
  // the second Q tile as a buffer of fp32 rows: 16-byte pieces per row (whole groups of eight) and rows that fit
  static constexpr int kMergePitch = (D / 4 + 7) / 8 * 8;
  static constexpr int kMergeRows = Base::kTileBytes / (16 * kMergePitch) < 128 ? 64 : 128;
  static_assert(kMergeRows * kMergePitch * 16 <= Base::kTileBytes, "merge buffer");
  // m, l of the rows in that buffer.  They have a place of their own: the second accumulator's warps may be segments ahead of the
  // reader (a pair of row tiles without keys waits for nothing) and store their output through the stage there.
  static constexpr int kMl = kStage + NQ * 4 * 4096;
  static constexpr int kBars = kMl + (NQ == 2 ? kMergeRows * 8 : 0);
  static constexpr int kUsed = kBars + 512 + kSegRing * (int)sizeof(ChunkSegment) + 1024;
  static constexpr int kTotal = kUsed < 116 * 1024 ? 116 * 1024 : kUsed;
};

// Has the phase completed?  Never suspends the thread (mbar_try_wait may, for microseconds).
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// A wait of the MMA and softmax warps, always true: one that expires (the status word then tells) sets `dead`, later ones do not
// last, and the warp leaves at its next segment, where all lanes look at it.  No vote and no way out of the loops in between: a
// vote per wait cost 80 cycles each, several times per key tile.
__device__ __forceinline__ bool chunk_wait(uint64_t* bar, uint32_t parity, const WaitCtx& ctx, bool& dead) {
  if (!mbar_try_wait(bar, parity) && !dead) dead = !mbar_wait(bar, parity, ctx);
  return true;
}

// tcgen05.mma with operand descriptors given as (lower, upper) halves; `accumulate` 0 starts the accumulator afresh.
__device__ __forceinline__ void tc_mma_ss32(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts32(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Row maximum of 128 scores in registers: eight chains.
__device__ __forceinline__ float row_max128(const uint32_t (&s)[128]) {
  float m[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) m[k] = __uint_as_float(s[k]);
#pragma unroll
  for (int i = 8; i < 128; i += 16)
#pragma unroll
    for (int k = 0; k < 8; ++k)
      m[k] = i + 8 + k < 128 ? max3(m[k], __uint_as_float(s[i + k]), __uint_as_float(s[i + 8 + k])) : fmaxf(m[k], __uint_as_float(s[i + k]));
  return max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
}

__device__ __forceinline__ void tmem_ld128(uint32_t taddr, uint32_t (&s)[128]) {
  uint32_t(&a)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[0]);
  uint32_t(&b)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[32]);
  uint32_t(&c)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[64]);
  uint32_t(&d)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[96]);
  tmem_ld32(taddr, a);
  tmem_ld32(taddr + 32, b);
  tmem_ld32(taddr + 64, c);
  tmem_ld32(taddr + 96, d);
}

// log2 of a common factor on P and the row sum.  fp16 loses weights below 2^-25, half of its smallest step, and over 128 Ki keys a
// 250th of the sum could go that way; weights reach 2^8 (the maximum may run that far ahead of its reference), so there is room for
// 2^7 more below 65504, and what is lost is below 2^-32 of the largest weight.  bf16 has the exponents of fp32.
template <typename T>
constexpr float kChunkWeightLift = Mma16816<T>::kSplitP ? 0.f : 7.f;

// P = exp2(s * scale - m_ref) of keys 64 h .. 64 h + 63 of one row, rounded to the input type, two keys to a register.  The
// row sum is taken before the rounding.  The special-function unit (16 per clock) needs 1024 cycles for the 128 x 128
// exponentials of a tile, as long as the tile's MMAs keep the tensor pipe.  (A part of them on the FMA pipe, as a polynomial of
// degree 3, was measured: one in eight gains 4 % of the cycles and nothing of the time, the clock gives way to the power limit;
// one in four or more loses.)
template <typename T>
__device__ __forceinline__ void chunk_exp_half(const uint32_t (&s)[128], int h, float scale_log2, float m_ref, uint32_t (&out)[32], float2 (&acc)[2]) {
  const float2 sc2 = make_float2(scale_log2, scale_log2), nm2 = make_float2(-m_ref, -m_ref);
#pragma unroll
  for (int w = 0; w < 32; ++w) {
    const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[64 * h + 2 * w]), __uint_as_float(s[64 * h + 2 * w + 1])), sc2, nm2);
    const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
    out[w] = Mma16816<T>::pack(e.x, e.y);
    acc[w & 1] = __fadd2_rn(acc[w & 1], e);
  }
}

// With the rounding residual tiles take a path of their own, in rolled loops of 32 columns over the scores in place.
// Maximum over the columns in [lo, hi]:
__device__ __forceinline__ float chunk_residual_max(uint32_t tS, int lo, int hi) {
  float m = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    uint32_t v[32];
    tmem_ld32(tS + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c + i >= lo && c + i <= hi) m = fmaxf(m, __uint_as_float(v[i]));
  }
  return m;
}
// ... and P: zero outside, the residual over the first 64 columns of the scores (never ahead of those still to be read).
// Returns the row sum.
template <typename T>
__device__ __forceinline__ float chunk_residual_exp(uint32_t tS, uint32_t tP, int lo, int hi, float scale_log2, float m_ref) {
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    uint32_t v[32], w[16], r[16];
    tmem_ld32(tS + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float a = c + i >= lo && c + i <= hi ? fast_exp2(fmaf(__uint_as_float(v[i]), scale_log2, -m_ref)) : 0.f;
      const float b = c + i + 1 >= lo && c + i + 1 <= hi ? fast_exp2(fmaf(__uint_as_float(v[i + 1]), scale_log2, -m_ref)) : 0.f;
      w[i / 2] = Mma16816<T>::pack(a, b);
      r[i / 2] = Mma16816<T>::pack_residual(a, b, w[i / 2]);
      sum += a + b;
    }
    tmem_st16(tP + c / 2, w);
    tmem_st16(tS + c / 2, r);
  }
  return sum;
}

// 1 / l for the row sum l: 0 for a row without keys, NaN where a score was not a number
__device__ __forceinline__ float chunk_inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }

// The 32 rows of a warp, one per lane in registers, to rows `row` (-1 = none) of `base` by way of `stage` (128 bytes per row):
// written as they are held, an instruction would write 16 bytes of 32 rows; from shared memory it writes contiguous bytes of a
// few.  EB = bytes per element; columns(c, x) gives columns [c * OC, (c + 1) * OC), pack(x) makes 16 bytes of them.
template <int D, int OC, int EB, typename Columns, typename Pack>
__device__ __forceinline__ void chunk_store_rows(unsigned char* stage, int lane, unsigned char* base, int row, const Columns& columns, const Pack& pack) {
  constexpr int kPieces = OC * EB / 16;  // 2, 4 or 8
  int to[kPieces];
#pragma unroll
  for (int it = 0; it < kPieces; ++it) to[it] = __shfl_sync(0xffffffffu, row, (it * 32 + lane) / kPieces);
  constexpr int kUnroll = EB == 2 && D / OC <= 2 ? 2 : 1;  // (the usual output goes straight through; the others are rolled)
#pragma unroll kUnroll
  for (int c = 0; c < D / OC; ++c) {
    float x[OC];
    columns(c, x);
#pragma unroll
    for (int k = 0; k < kPieces; ++k) *reinterpret_cast<uint4*>(stage + lane * 128 + ((k ^ (lane & 7)) << 4)) = pack(x + k * (16 / EB));
    __syncwarp();
    uint4 v[kPieces];
#pragma unroll
    for (int it = 0; it < kPieces; ++it) {
      const int r = (it * 32 + lane) / kPieces, piece = (it * 32 + lane) % kPieces;
      v[it] = *reinterpret_cast<const uint4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
    }
#pragma unroll
    for (int it = 0; it < kPieces; ++it) {
      const int piece = (it * 32 + lane) % kPieces;
      if (to[it] >= 0) *reinterpret_cast<uint4*>(base + (size_t)to[it] * (D * EB) + (c * kPieces + piece) * 16) = v[it];
    }
    __syncwarp();
  }
}

// Adds the values that are not finite and were zeroed for other rows' sake to the stored row of token `tok` of the item and head `head`
// of the tile, where it sees their keys.  A rare path, so a function of its own: inlined, its registers cost the hot loop 60 bytes of
// spills and chunks of a prompt 1.4 %.
template <typename T, int D, int TPP>
__device__ __noinline__ void chunk_add_bad_values(const ChunkParams& p, const ChunkSegment& g, int tok, int head) {
  const int pos = g.pos0 + tok;
  const int hi = p.causal ? min(pos, g.key_cap - 1) : g.key_cap - 1, lo = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
  const bool direct = g.slot < 0, f32 = !direct || p.out_f32;
  const size_t at = (direct ? (size_t)(g.row0 + tok) * p.num_q_heads + g.head0 + head : (size_t)g.slot * p.part_rows + tok * p.tile_heads + head) * D;
  float* out32 = (direct ? static_cast<float*>(p.out) : p.part_acc) + at;
  T* out16 = static_cast<T*>(p.out) + at;
#pragma unroll 1
  for (int k = 0; k < 96; ++k) {  // groups of eight keys, which the V pool keeps side by side
    uint32_t left = (g.bad[k >> 4][(k >> 2) & 3] >> ((k & 3) * 8)) & 0xffu;
    if (left == 0) continue;
    const int key0 = ((k < 48 ? g.some_hi / kTile : g.key_lo / kTile - 3) + (k >> 4)) * kTile + (k & 15) * 8;
    if (key0 < lo) left &= 0xffu << min(lo - key0, 8);
    if (key0 + 7 > hi) left &= 0xffu >> min(key0 + 7 - hi, 8);
    if (left == 0) continue;
    const long long page = min((long long)p.page_table[(size_t)g.seq * p.max_pages_per_seq + key0 / TPP], p.num_pages - 1);
    const T* v = static_cast<const T*>(p.v_pool) + ((size_t)page * p.num_kv_heads + g.kv_head) * (D * TPP) + key0 % TPP;
    int nans = 0;
#pragma unroll 1
    for (int d0 = 0; d0 < D; d0 += 4) {
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint4*>(v + (d0 + i) * TPP);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        float sum = 0.f;
        bool found = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 pair = Mma16816<T>::unpack(w[e >> 1]);
          const float f = e & 1 ? pair.y : pair.x;
          if ((left >> e & 1) && !isfinite(f)) {
            sum += f;
            found = true;
          }
        }
        if (!found) continue;
        nans += isnan(sum);
        if (f32)
          out32[d0 + i] += sum;
        else
          out16[d0 + i] = Mma16816<T>::from_float(Mma16816<T>::to_float(out16[d0 + i]) + sum);
      }
    }
    if (nans == D) return;  // (whole tokens that are not numbers: nothing changes the row any more)
  }
}

template <typename T, int D, int TPP, int NQ>
__global__ void __launch_bounds__(128 + 128 * NQ, 1)
    chunk_tcgen05_kernel(const __grid_constant__ ChunkParams p, const __grid_constant__ CUtensorMap tm_q,
                         const __grid_constant__ CUtensorMap tm_vpool) {
  using C = ChunkCfg<D, TPP, NQ>;
  using B = typename C::Base;
  constexpr int ST = C::ST, NS = C::kSBuffers, kThreadsAll = C::kThreads;
  constexpr int kBlocks = B::kBlocks, kPagesPerTile = B::kPagesPerTile, kPageBytes = B::kPageBytes, kTileBytes = B::kTileBytes;
  constexpr int kOC = B::kOChunk;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = smem + C::kQ;
  unsigned char* sK = smem + C::kK;
  unsigned char* sV = smem + C::kV;
  float2* sMl = reinterpret_cast<float2*>(smem + C::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* q_full = bars;             // 1
  uint64_t* q_empty = bars + 1;        // 1: the last QK^T of a segment has read Q
  uint64_t* merge_full = bars + 2;     // 1: the second accumulator's rows are in shared memory
  uint64_t* merge_empty = bars + 3;    // 1
  uint64_t* s_full = bars + 6;         // 2, per accumulator: its scores are in an S buffer
  uint64_t* s_empty = bars + 8;        // 2: ... and have been read
  uint64_t* p_full = bars + 10;        // 2: its P tile is written
  uint64_t* o_done = bars + 12;        // 2: the PV that read it has run
  uint64_t* k_full = bars + 14;        // ST
  uint64_t* k_empty = bars + 18;       // ST
  uint64_t* v_full = bars + 22;        // ST
  uint64_t* v_empty = bars + 26;       // ST
  uint64_t* seg_full = bars + 30;      // kSegRing
  uint64_t* seg_empty = bars + 34;     // kSegRing
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 38);
  long long* sm_plan = reinterpret_cast<long long*>(bars + 40);  // scan scratch, then the share's last item
  ChunkSegment* segs = reinterpret_cast<ChunkSegment*>(smem + C::kBars + 512);
  static_assert(kSegRing == 4 && ST <= 4 && kThreadsAll / 32 <= 12, "barrier layout");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int item_tokens = NQ * p.tile_tokens;
  auto item_cost = [&](const ChunkSeq& q, int ta) {
    const ChunkCost c = chunk_cost<T, D, NQ>(p, q, ta);
    int lo, hi;
    return c.setup + c.tile * chunk_keys(p, q, ta, min(ta + item_tokens, q.n), lo, hi);
  };
  const int vheads = p.num_kv_heads * p.head_blocks;

  // ---- the CTA's share of the line of items ----
  // thread t sums the cost of a run of sequences; one scan places the runs on the line
  long long share0, share1;
  {
    const int per = (p.num_seqs + kThreadsAll - 1) / kThreadsAll;
    const int sa = min(tid * per, p.num_seqs), sb = min(sa + per, p.num_seqs);
    long long mine = 0;
    int least = kChunkMinShare;
    for (int s = sa; s < sb; ++s) {
      const ChunkSeq q = chunk_seq(p, s, TPP);
      long long w = 0;
      for (int ta = 0; ta < q.n; ta += item_tokens) {
        w += item_cost(q, ta);
        least = max(least, chunk_cost<T, D, NQ>(p, q, ta).tile);
      }
      mine += w * vheads;
    }
    long long inc = mine;
#pragma unroll
    for (int sh = 1; sh < 32; sh <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, sh);
      if (lane >= sh) inc += up;
    }
    least = __reduce_max_sync(0xffffffffu, least);
    if (lane == 31) {
      sm_plan[warp] = inc;
      sm_plan[12 + warp] = least;
    }
    if (tid == 0) {
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      for (int i = 0; i < ST; ++i) {
        mbar_init(&k_full[i], 32);
        mbar_init(&k_empty[i], 1);
        mbar_init(&v_full[i], 1);
        mbar_init(&v_empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 4);
        mbar_init(&s_empty[i], 4);
        mbar_init(&o_done[i], 1);
      }
      mbar_init(merge_full, 4);
      mbar_init(merge_empty, 4);
      for (int i = 0; i < kSegRing; ++i) {
        mbar_init(&seg_full[i], 1);
        mbar_init(&seg_empty[i], 3 + 4 * NQ);
      }
      fence_mbar_init();
    }
    if (warp == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kThreadsAll / 32; ++w) {
      const long long v = sm_plan[w];
      if (w < warp) before += v;
      total += v;
      least = max(least, (int)sm_plan[12 + w]);
    }
    const long long share = max((total + gridDim.x - 1) / gridDim.x, (long long)least);
    share0 = min(share * blockIdx.x, total);
    share1 = min(share0 + share, total);
    __syncthreads();
    const long long start = before + inc - mine;
    const long long last = share1 - 1;
    if (share0 < share1 && last >= start && last < start + mine) {
      // the share ends in this thread's run: find the item
      long long at = start;
      int s = sa, vh = 0, ta = 0;
      for (; s < sb; ++s) {
        const ChunkSeq q = chunk_seq(p, s, TPP);
        long long w = 0;
        for (int t = 0; t < q.n; t += item_tokens) w += item_cost(q, t);
        if (last < at + w * vheads) {
          vh = (int)((last - at) / w);
          at += vh * w;
          for (;; ta += item_tokens) {
            const int c = item_cost(q, ta);
            if (last < at + c) break;
            at += c;
          }
          break;
        }
        at += w * vheads;
      }
      sm_plan[0] = s;
      sm_plan[1] = vh;
      sm_plan[2] = ta;
      sm_plan[3] = at;
      sm_plan[4] = share;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // With two accumulators three warpgroups start with 168 registers a thread (384 x 168 = 64512 of the SM's 65536); the
  // softmax warpgroups hold a row of 128 scores each and take 216, which the first one leaves them: 128 x 72 + 256 x 216 = 64512.
  if (warp < 4) {
  if (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 0) {
    // =============================== segments, Q and V ===============================
    if (share0 >= share1) {
      if (lane == 0) p.cuts[blockIdx.x].parts = 0;
    }
    // The share is walked backwards.  What it holds of its last item are that item's first keys, and what it holds of its
    // first item that item's last ones: so all CTAs start at the first keys and end at the last, and row tiles of one head,
    // which lie on neighbouring CTAs, read the same pages at about the same time (from L2, when one sequence is larger).
    int s = 0, vh = 0, ta = 0;
    long long at = 0, share = 1;  // at: where the current item starts
    bool more = share0 < share1;
    if (more) {
      s = (int)sm_plan[0];
      vh = (int)sm_plan[1];
      ta = (int)sm_plan[2];
      at = sm_plan[3];
      share = sm_plan[4];
    }
    __syncwarp();
    ChunkSeq q = more ? chunk_seq(p, s, TPP) : ChunkSeq{};
    int lo = 0, hi = 0, nt = more ? chunk_keys(p, q, ta, min(ta + item_tokens, q.n), lo, hi) : 0;
    uint32_t n_pub = 0;  // segments published (ring position)
    bool cut_written = false;
    // next segment of the share (the same computation on every lane), published to the other warps
    auto publish = [&]() {
      // ---- next segment of the share (the same computation on every lane) ----
      ChunkWork g;
      g.end = 1;
      while (more && g.end) {
        // a key tile belongs to the share that its place on the line starts in
        const ChunkCost cost = chunk_cost<T, D, NQ>(p, q, ta);
        const long long first = at + cost.setup;
        auto tiles_before = [&](long long x) {
          const int d = (int)min(max(x - first, 0LL), (long long)nt * cost.tile);  // (a tile count of an int32 length, times 14 at most)
          return (d + cost.tile - 1) / cost.tile;
        };
        const int t0 = tiles_before(share0), t1 = tiles_before(share1);
        if (t1 > t0 || (nt == 0 && at >= share0)) {
          g.end = 0;
          g.seq = s;
          g.kv_head = vh / p.head_blocks;
          const int hb = vh - g.kv_head * p.head_blocks;
          g.head0 = g.kv_head * p.group + hb * p.tile_heads;
          g.heads = min(p.tile_heads, p.group - hb * p.tile_heads);
          g.row0 = q.row0 + ta;
          g.tokens = min(item_tokens, q.n - ta);
          g.pos0 = q.len - q.n + ta;
          g.kt0 = lo / kTile + t0;
          g.kt1 = lo / kTile + t1;
          g.key_lo = lo;
          g.key_hi = hi;
          g.key_cap = q.cap;
          g.some_hi = p.causal ? max(lo, min(hi, g.pos0 + 1)) : hi;
          g.some_lo = p.window > 0 ? min(hi, max(lo, g.pos0 + g.tokens - p.window)) : lo;
          g.any_bad = 0;
          g.alternate = NQ == 2 && g.tokens <= p.tile_tokens;
          g.residual = chunk_feeds_residual<T>(p, q, ta);
          g.slot = t0 > 0 ? 2 * (int)blockIdx.x : (t1 < nt ? 2 * (int)blockIdx.x + 1 : -1);
          if (t0 == 0 && t1 < nt && lane == 0) {
            // this CTA holds the item's first part: tell the merging kernel where the others are
            ChunkCut c;
            c.parts = (int)((first + (long long)(nt - 1) * cost.tile) / share) - (int)blockIdx.x + 1;
            c.row0 = g.row0;
            c.tokens = g.tokens;
            c.head0 = g.head0;
            c.heads = g.heads;
            p.cuts[blockIdx.x] = c;
            cut_written = true;
          }
        }
        // back to the item before, if the share reaches it: row tiles, then heads, then sequences
        more = at > share0;
        if (!more) break;
        if (ta > 0) {
          ta -= item_tokens;
        } else {
          if (--vh < 0) {
            vh = vheads - 1;
            do q = chunk_seq(p, --s, TPP);
            while (q.n <= 0);  // (an item lies before this one: at > 0)
          }
          ta = (q.n - 1) / item_tokens * item_tokens;
        }
        nt = chunk_keys(p, q, ta, min(ta + item_tokens, q.n), lo, hi);
        at -= item_cost(q, ta);
      }
      const int slot = n_pub % kSegRing;
      if (!__all_sync(0xffffffffu, mbar_wait(&seg_empty[slot], ((n_pub / kSegRing) & 1) ^ 1, p.status))) return false;
      if (lane < 24) segs[slot].bad[lane >> 2][lane & 3] = 0u;
      __syncwarp();
      if (lane == 0) {
        static_cast<ChunkWork&>(segs[slot]) = g;
        mbar_arrive(&seg_full[slot]);
      }
      __syncwarp();
      ++n_pub;
      return true;
    };
    uint32_t n_tile = 0;
    bool prev_alternate = false;
    int ok = publish();
    for (uint32_t n_seg = 0; ok; ++n_seg) {
      const ChunkSegment& g = segs[n_seg % kSegRing];  // (not overwritten before three more are published)
      const int end = g.end, kt0 = g.kt0, kt1 = g.kt1, alternate = g.alternate;
      if (end) break;
      // ---- Q: free once the last QK^T of the previous segment has run; the second tile also serves as the merge buffer of
      // alternate segments ----
      if (lane == 0) {
        ok = mbar_wait(q_empty, (n_seg & 1) ^ 1, p.status);
        // (QK^T runs up to two segments ahead of the softmax, so a barrier that counts segments could be two phases behind
        // and its parity mistaken; the previous segment's slot cannot be released twice before its ring comes round)
        if (ok && !alternate && prev_alternate) ok = mbar_wait(&seg_empty[(n_seg - 1) % kSegRing], ((n_seg - 1) / kSegRing) & 1, p.status);
        if (ok && kt0 < kt1) {
          const int tiles = NQ == 2 && !alternate ? 2 : 1;
          mbar_arrive_expect_tx(q_full, tiles * kBlocks * p.tile_heads * p.tile_tokens * 128);
          for (int t = 0; t < tiles; ++t)
            for (int kb = 0; kb < kBlocks; ++kb)
              tma_load_3d(sQ + t * kTileBytes + kb * kBlockBytes, &tm_q, kb * 64, g.head0, g.row0 + t * p.tile_tokens, q_full);
        } else if (ok) {
          mbar_arrive(q_full);  // no keys: the segment only passes through the barriers that count segments
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      prev_alternate = alternate != 0;
      // (the next segment is announced before this one's V tiles, so that its K can be on the way)
      if (ok) ok = publish();
      // ---- V ----
      const int key_lo = g.key_lo, key_hi = g.key_hi, kv_head = g.kv_head;
      const uint32_t* pages = p.page_table + (size_t)g.seq * p.max_pages_per_seq;
      for (int j = kt0; j < kt1 && ok; ++j, ++n_tile) {
        const int st = n_tile % ST;
        const int pg0 = max(0, key_lo - j * kTile) / TPP, pg1 = (min(kTile, key_hi - j * kTile) + TPP - 1) / TPP;
        uint32_t pid = 0;
        if (lane >= pg0 && lane < pg1) {
          pid = pages[j * kPagesPerTile + lane];
          if ((long long)pid >= p.num_pages) pid = (uint32_t)(p.num_pages - 1);
        }
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], ((n_tile / ST) & 1) ^ 1, p.status)))) break;
        if (lane == 0) mbar_arrive_expect_tx(&v_full[st], (pg1 - pg0) * kPageBytes);
        __syncwarp();
        if (lane >= pg0 && lane < pg1)
          tma_load_3d(sV + st * kTileBytes + lane * kPageBytes, &tm_vpool, 0, 0, (int)(pid * p.num_kv_heads + kv_head), &v_full[st]);
      }
    }
    if (lane == 0 && share0 < share1 && !cut_written) p.cuts[blockIdx.x].parts = 0;
  } else if (warp == 1 || warp == 2) {
    // =============================== MMA issuers: QK^T and PV ===============================
    // A segment is a list of steps, one per (key tile, accumulator).  QK^T of step k goes into the S buffer as soon as the
    // softmax warps have read the scores before it (into registers: a step's QK^T runs under the softmax of the step
    // before it), PV of step k when its P is there.  The two share nothing but barriers, so each has a warp: one warp that
    // issues both spends more time on the issue (8 MMAs, waits and commits: ~600 cycles each) than the MMAs take.
    constexpr int F = Fmt<T>::kCode;
    bool dead = false;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return chunk_wait(bar, parity, p.status, dead); };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) tc_commit(bar);
    };
    // (broadcast: the issuing code is warp-uniform, which the compiler cannot know of values from shared memory)
    auto uniform = [&](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const bool is_qk = warp == 1;
    uint32_t n_seg = 0;
    uint32_t n_tile = 0;            // key tiles whose last MMA has been issued
    uint32_t n_a0 = 0, n_a1 = 0;    // steps of each accumulator so far
    int last_acc = -1;              // whose scores the single S buffer holds
    bool ok = true;
    while (ok) {
      const int slot = n_seg % kSegRing;
      wait_all(&seg_full[slot], (n_seg / kSegRing) & 1);
      if (__any_sync(0xffffffffu, dead)) break;
      const ChunkSegment& sg = segs[slot];
      const int end = uniform(sg.end), kt0 = uniform(sg.kt0), num = uniform(sg.kt1) - kt0, key_lo = uniform(sg.key_lo), key_hi = uniform(sg.key_hi);
      const int pair = NQ == 2 && !uniform(sg.alternate) ? 1 : 0;
      const bool residual = Mma16816<T>::kSplitP && uniform(sg.residual);
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[slot]);
      if (end) break;
      ++n_seg;
      const int steps = pair ? 2 * num : num;
      if (is_qk) {
        constexpr uint32_t idesc_qk = make_idesc(128, F, F, 0);
        // An operand's descriptor is its constant upper half and (address >> 4) plus a constant: 32-bit arithmetic per MMA.
        constexpr uint32_t hi_q = (1024u >> 4) | (1u << 14) | (uint32_t)(kLayoutSw128 << 29);
        constexpr uint32_t hi_k = (128u >> 4) | (1u << 14) | (uint32_t)(kLayoutNone << 29);
        const uint32_t lo_q = (smem_u32(sQ) >> 4) | (1u << 16);
        const uint32_t lo_k = (smem_u32(sK) >> 4) | ((B::kChunkBytes >> 4) << 16);
        ok = wait_all(q_full, (n_seg - 1) & 1);
        if (ok && num <= 0 && lane == 0) mbar_arrive(q_empty);
        for (int k = 0; k < steps && ok; ++k) {
          const int acc = NQ == 2 ? k & 1 : 0, st = n_tile % ST;
          // the buffer's previous scores have been read
          const int user = NS == 2 ? acc : last_acc;
          const uint32_t uses = user == 1 ? n_a1 : n_a0;
          if (user >= 0 && uses > 0 && !(ok = wait_all(&s_empty[user], (uses - 1) & 1))) break;
          if ((!pair || acc == 0) && !(ok = wait_all(&k_full[st], (n_tile / ST) & 1))) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + (NS == 2 ? acc * kTile : 0), a = lo_q + (pair ? acc : 0) * (kTileBytes >> 4), b = lo_k + st * (kTileBytes >> 4);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              tc_mma_ss32(d_tmem, a + (((ks >> 2) * kBlockBytes + (ks & 3) * 32) >> 4), hi_q, b + ((ks * 2 * B::kChunkBytes) >> 4), hi_k, idesc_qk, ks > 0);
            tc_commit(&s_full[acc]);
            if (!pair || acc == 1) tc_commit(&k_empty[st]);
            if (k == steps - 1) tc_commit(q_empty);
          }
          __syncwarp();
          if (acc) ++n_a1; else ++n_a0;
          last_acc = acc;
          if (!pair || acc == 1) ++n_tile;
        }
      } else {
        constexpr uint32_t idesc_pv = make_idesc(D, F, F, 0);
        constexpr uint32_t hi_v = ((8u * TPP * 2) >> 4) | (1u << 14) | (uint32_t)((TPP == 16 ? kLayoutSw32 : kLayoutSw64) << 29);
        const uint32_t lo_v = (smem_u32(sV) >> 4) | (1u << 16);
        constexpr auto off = [](int kk) { return (TPP == 16 ? kk * kPageBytes : (kk >> 1) * kPageBytes + (kk & 1) * 32) >> 4; };
        for (int k = 0; k < steps && ok; ++k) {
          const int acc = NQ == 2 ? k & 1 : 0, st = n_tile % ST, i = pair ? k >> 1 : k, j = kt0 + i;
          const int kk0 = max(0, key_lo - j * kTile) >> 4, kk1 = (min(kTile, key_hi - j * kTile) + 15) >> 4;  // 16-key steps in use
          const uint32_t fresh = (pair ? i == 0 : k < NQ) ? 1 : 0;                                            // the accumulator starts here
          if ((!pair || acc == 0) && !(ok = wait_all(&v_full[st], (n_tile / ST) & 1))) break;
          if (!(ok = wait_all(&p_full[acc], (acc ? n_a1 : n_a0) & 1))) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + C::kOCol + acc * B::DP, a = tmem_base + C::kPCol + acc * 64, b = lo_v + st * (kTileBytes >> 4);
          if (elect_one()) {
            if (kk0 == 0 && kk1 == kTile / 16) {
              tc_mma_ts32(d_tmem, a, b, hi_v, idesc_pv, !fresh);
#pragma unroll
              for (int kk = 1; kk < kTile / 16; ++kk) tc_mma_ts32(d_tmem, a + kk * 8, b + off(kk), hi_v, idesc_pv, 1);
            } else {
#pragma unroll 1
              for (int kk = kk0; kk < kk1; ++kk) tc_mma_ts32(d_tmem, a + kk * 8, b + off(kk), hi_v, idesc_pv, !(fresh && kk == kk0));
            }
            if (residual) {
              const uint32_t r = tmem_base + (NS == 2 ? acc * kTile : 0);
#pragma unroll 1
              for (int kk = kk0; kk < kk1; ++kk) tc_mma_ts32(d_tmem, r + kk * 8, b + off(kk), hi_v, idesc_pv, 1);
            }
            tc_commit(&o_done[acc]);
            if (!pair || acc == 1) tc_commit(&v_empty[st]);
          }
          __syncwarp();
          if (acc) ++n_a1; else ++n_a0;
          if (!pair || acc == 1) ++n_tile;
        }
      }
    }
  } else {
    // =============================== K ===============================
    // K comes by 16-byte asynchronous copies, lane = token: a page keeps the tokens of a chunk in a row, so 32 lanes write 512
    // contiguous bytes and read two page rows.  (A TMA gather of four page rows per request brings the same tile in 2590
    // cycles, these copies in less than 1200, the turn-around of the ring it was measured with.)
    uint32_t n_seg = 0, n_tile = 0;
    uint32_t handed = 0;  // tiles whose copies have landed and been handed over (n_tile: whose copies have been issued)
    bool ok = true;
    // hands over every tile but the newest KEEP
    auto hand_over = [&](auto keep) {
      constexpr uint32_t KEEP = decltype(keep)::value;
      if (n_tile - handed <= KEEP) return;
      asm volatile("cp.async.wait_group %0;" ::"n"(KEEP) : "memory");  // (a tile is a group of copies)
      fence_proxy_async_smem();                                       // (read by MMAs)
#pragma unroll 1
      for (; n_tile - handed > KEEP; ++handed) mbar_arrive(&k_full[handed % ST]);
    };
    // a wait that may last hands over first what may be waited for
    auto wait_stage = [&](uint64_t* bar, uint32_t parity) {
      if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
      hand_over(std::integral_constant<int, 0>());
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)) != 0;
    };
    while (ok) {
      const int slot = n_seg % kSegRing;
      if (!(ok = wait_stage(&seg_full[slot], (n_seg / kSegRing) & 1))) break;
      const int end = segs[slot].end, kt0 = segs[slot].kt0, kt1 = segs[slot].kt1, key_lo = segs[slot].key_lo, key_hi = segs[slot].key_hi;
      const int kv_head = segs[slot].kv_head;
      const uint32_t* pages = p.page_table + (size_t)segs[slot].seq * p.max_pages_per_seq;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[slot]);
      if (end) {
        hand_over(std::integral_constant<int, 0>());
        break;
      }
      ++n_seg;
      // pages [first, last] of key tile j hold visible keys; the others are not touched (their columns of S are masked)
      auto first_page = [&](int j) { return max(0, key_lo - j * kTile) / TPP; };
      auto last_page = [&](int j) { return (min(kTile, key_hi - j * kTile) - 1) / TPP; };
      auto page_id = [&](int j) {  // lane l: the id of page l of the tile (of the nearest one in use)
        uint32_t pid = 0;
        if (lane < kPagesPerTile && j < kt1) {
          pid = pages[j * kPagesPerTile + min(max(lane, first_page(j)), last_page(j))];
          if ((long long)pid >= p.num_pages) pid = (uint32_t)(p.num_pages - 1);
        }
        return pid;
      };
      uint32_t next_pid = page_id(kt0);
      for (int j = kt0; j < kt1; ++j) {
        const int st = n_tile % ST;
        const uint32_t pid = next_pid;
        next_pid = page_id(j + 1);
        const int pg0 = first_page(j), pg1 = last_page(j) + 1;
        if (!(ok = wait_stage(&k_empty[st], ((n_tile / ST) & 1) ^ 1))) break;
        const uint32_t k_dst = smem_u32(sK) + st * kTileBytes + lane * 16;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          const int tok = q * 32 + lane, pg = tok / TPP;
          const uint32_t id = __shfl_sync(0xffffffffu, pid, pg);
          const unsigned char* src = static_cast<const unsigned char*>(p.k_pool) + ((size_t)id * p.num_kv_heads + kv_head) * kPageBytes + (tok % TPP) * 16;
          if (pg >= pg0 && pg < pg1)
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(k_dst + q * 512 + c * B::kChunkBytes), "l"(src + c * (TPP * 16)) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++n_tile;
        hand_over(std::integral_constant<int, (ST > 2 ? ST - 1 : 1)>());
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  } else {
    if (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // =============================== softmax warpgroups ===============================
    const int wg = (warp - 4) >> 2;
    const int lane_group = warp & 3;
    const int row = lane_group * 32 + lane;
    unsigned char* stage = smem + C::kStage + (warp - 4) * 4096;
    const uint32_t lane_addr = (uint32_t)(lane_group * 32) << 16;
    const uint32_t tO = tmem_base + lane_addr + C::kOCol + wg * B::DP, tP = tmem_base + lane_addr + C::kPCol + wg * 64;
    const uint32_t tS = tmem_base + lane_addr + (NS == 2 ? wg * kTile : 0);
    bool dead = false;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return chunk_wait(bar, parity, p.status, dead); };
    uint32_t n_seg = 0, n_s = 0, n_o = 0, n_v = 0, n_merge = 0;  // segments, scores taken, PVs seen to end, key tiles, merges
    bool ok = true;
    while (ok) {
      const int slot = n_seg % kSegRing;
      wait_all(&seg_full[slot], (n_seg / kSegRing) & 1);
      if (__any_sync(0xffffffffu, dead)) break;
      ChunkSegment& g = segs[slot];  // (held until the segment is done: what the epilogue needs stays in shared memory)
      if (g.end) break;
      ++n_seg;
      const bool alt = NQ == 2 && g.alternate;
      const int q_tile = alt ? 0 : wg;                   // which tile of rows this accumulator holds
      const int tok = row / p.tile_heads;                // of the tile
      const int head = row - tok * p.tile_heads;
      const int tok_first = q_tile * p.tile_tokens;      // the tile's first token in the item
      const int tile_tokens = max(0, min(p.tile_tokens, g.tokens - tok_first));
      const bool row_exists = tok < tile_tokens && head < g.heads;
      const bool warp_works = (lane_group * 32) / p.tile_heads < tile_tokens;  // some row of the warp may exist
      // keys this row sees: [lo, hi]
      const int pos = g.pos0 + tok_first + tok;
      const int hi = p.causal ? min(pos, g.key_cap - 1) : g.key_cap - 1;
      const int lo = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
      // ... and the keys that all rows of this warp see, [all_lo, all_hi]
      const int pos_a = g.pos0 + tok_first + lane_group * 32 / p.tile_heads, pos_b = g.pos0 + tok_first + (lane_group * 32 + 31) / p.tile_heads;
      const int all_hi = p.causal ? min(pos_a, g.key_cap - 1) : g.key_cap - 1;
      const int all_lo = p.window > 0 && pos_b >= p.window ? pos_b - p.window + 1 : 0;
      const bool residual = Mma16816<T>::kSplitP && g.residual;
      // (rows that do not exist hold other tokens' queries or whatever was there: with an infinite maximum they never ask for a
      // rescaling, whose rounding would differ from call to call)
      float m_used = row_exists ? -INFINITY : INFINITY, l_run = 0.f;
      const int kt0 = g.kt0, num = g.kt1 - kt0;
      // key tiles with values that not all rows see: up to `care_lo`, and from `care_hi` on
      const int care_lo = g.key_lo & 15 || g.some_lo > g.key_lo ? (max(g.some_lo, g.key_lo + 1) - 1) / kTile : -1;
      const int care_hi = g.some_hi < g.key_hi ? g.some_hi / kTile : g.key_hi & 15 ? g.key_hi / kTile : 0x7fffffff;
      int mine = 0;  // key tiles this accumulator has taken
      for (int i = 0; i < num; ++i) {
        if (alt && (i & 1) != wg) {
          ++n_v;
          continue;
        }
        const int j = kt0 + i;
        if (!(ok = wait_all(&s_full[wg], n_s & 1))) break;
        ++n_s;
        tc_fence_after();
        auto scores_read = [&]() {  // (behind a warp-wide tcgen05 wait)
          tc_fence_before();
          if (lane == 0) mbar_arrive(&s_empty[wg]);
        };
        // O and the P tile are this warp's again once the PV of the previous key tile has run
        bool pv_done = mine == 0 || residual;
        auto wait_pv = [&]() {
          if (!pv_done) {
            if (!wait_all(&o_done[wg], n_o & 1)) return false;
            ++n_o;
            tc_fence_after();
            pv_done = true;
          }
          return true;
        };
        // Values that a row does not see are multiplied by P = 0, which is not 0 if they hold an infinity or a NaN.  So, in the
        // 16-key steps that are used: slots that no row of the item sees (past the last key, before the window, never written)
        // are zeroed; a value that some rows see and others do not is zeroed if it is not finite, and its key noted: the rows
        // that see it have it added to their output.  (Values that all rows see need no care.)
        auto clear_values = [&]() {
          const int c_lo = max(0, g.key_lo - j * kTile), c_hi = min(kTile, g.key_hi - j * kTile);
          const int some_lo = g.some_lo - j * kTile, some_hi = g.some_hi - j * kTile;
          const int st = (int)(n_v % ST);
          if (!wait_all(&v_full[st], (n_v / ST) & 1)) return false;
          unsigned char* vt = sV + st * kTileBytes;
          constexpr uint32_t kAbs = 0x7fff7fffu, kCarry = Mma16816<T>::kSplitP ? 0x00800080u : 0x04000400u;  // bf16, fp16
          const int first = c_lo & ~15, last = (c_hi + 15) & ~15;  // (multiples of 8)
          for (int dr = row; dr < D; dr += 128) {
            const int sw = TPP == 16 ? ((dr >> 2) & 1) : ((dr >> 1) & 3);
#pragma unroll 1
            for (int c = first; c < last; c += 8) {
              const bool edge = c < c_lo || c + 8 > c_hi;
              if (!edge && c >= some_lo && c + 8 <= some_hi) continue;  // seen by all rows
              uint4* at = reinterpret_cast<uint4*>(vt + (c / TPP) * kPageBytes + dr * (TPP * 2) + ((((c % TPP) >> 3) ^ sw) << 4));
              uint32_t w[4] = {at->x, at->y, at->z, at->w};
              // (a magnitude with all exponent bits set carries into the sign bit)
              const uint32_t off = (((w[0] & kAbs) + kCarry) | ((w[1] & kAbs) + kCarry) | ((w[2] & kAbs) + kCarry) | ((w[3] & kAbs) + kCarry)) & 0x80008000u;
              if (!edge && !off) continue;
#pragma unroll 1
              for (int e = 0; e < 8; ++e) {
                const int col = c + e;
                const uint32_t mask = 0xffffu << ((e & 1) * 16);
                const bool seen = col >= c_lo && col < c_hi;
                const uint32_t word = e < 2 ? w[0] : e < 4 ? w[1] : e < 6 ? w[2] : w[3];
                const bool finite = !(((word & kAbs) + kCarry) & 0x80008000u & mask);
                if (seen && (finite || (col >= some_lo && col < some_hi))) continue;
                if (seen) {
                  const int key = j * kTile + col, d0 = g.some_hi / kTile;
                  atomicOr(&g.bad[key >= g.some_hi ? j - d0 : 3 + j - g.key_lo / kTile][col >> 5], 1u << (col & 31));
                  g.any_bad = 1;
                }
                const uint32_t kept = word & ~mask;
                if (e < 2) w[0] = kept; else if (e < 4) w[1] = kept; else if (e < 6) w[2] = kept; else w[3] = kept;
              }
              *at = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          fence_proxy_async_smem();
          return true;
        };
        // takes the row maximum of this tile in; the caller has scaled it (scale > 0: the maximum commutes with the scaling)
        auto new_max = [&](float mx) {
          const float m_new = fmaxf(m_used, mx);
          if (mine == 0) {
            m_used = m_new;
          } else if (__any_sync(0xffffffffu, m_new > m_used + kRescaleThreshold)) {
            if (!wait_pv()) return false;
            const float f = m_new > m_used ? fast_exp2(m_used - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < D / kOC; ++c) {
              uint32_t v[kOC];
              tmem_ldw(tO + c * kOC, v);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < kOC; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
              tmem_stw(tO + c * kOC, v);
            }
            l_run *= f;
            m_used = m_new;
          }
          return true;
        };
        // One tile without residual: the row in registers, straight through.  (One path for masked tiles and others, and little
        // control flow in it: masking group by group, with a branch each, made the compiler spill the scores, at twice the time
        // of every tile; a masked copy of the path costs 5 % through the instruction cache.)
        auto plain_tile = [&](bool masked, int rl, int rh) {
          uint32_t sc[128];
          tmem_ld128(tS, sc);
          tmem_wait_ld();
          scores_read();
          if (masked) {
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (c > rh) sc[c] = 0xff800000u;
            if (rl > 0) {
#pragma unroll
              for (int c = 0; c < 128; ++c)
                if (c < rl) sc[c] = 0xff800000u;
            }
          }
          if (!new_max(row_max128(sc) * p.scale_log2)) return false;
          const float m_ref = (m_used > -INFINITY ? m_used : 0.f) - kChunkWeightLift<T>;
          float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          uint32_t w[32];
          chunk_exp_half<T>(sc, 0, p.scale_log2, m_ref, w, acc);
          if (!wait_pv()) return false;
          tmem_st32(tP, w);
          chunk_exp_half<T>(sc, 1, p.scale_log2, m_ref, w, acc);
          tmem_st32(tP + 32, w);
          l_run += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
          tmem_wait_st();
          return true;
        };
        if (!warp_works) {
          if (!residual) scores_read();
          if (!(ok = wait_pv())) break;
        } else if (residual) {
          const int rl = lo - j * kTile, rh = hi - j * kTile;
          if (!(ok = new_max(chunk_residual_max(tS, rl, rh) * p.scale_log2) && wait_pv())) break;
          l_run += chunk_residual_exp<T>(tS, tP, rl, rh, p.scale_log2, m_used > -INFINITY ? m_used : 0.f);
          tmem_wait_st();  // (the score buffer now holds the residual, and is given back after the PV)
        } else {
          const int c0 = j * kTile;
          ok = plain_tile(c0 < all_lo || c0 + kTile - 1 > all_hi, lo - c0, hi - c0);
          if (!ok) break;
        }
        ++mine;
        if ((wg == 0 || alt) && (j <= care_lo || j >= care_hi) && !(ok = clear_values())) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[wg]);
        if (residual) {
          // (the S buffer holds the residual until the PV has run)
          if (!(ok = wait_all(&o_done[wg], n_o & 1))) break;
          ++n_o;
          scores_read();
        }
        ++n_v;
      }
      if (!ok) break;
      // ---- epilogue ----
      // O is complete once the last PV has run
      if (mine > 0 && !residual) {
        ok = wait_all(&o_done[wg], n_o & 1);
        ++n_o;
        if (!ok) break;
      }
      tc_fence_after();
      // (a row whose keys here are all NaN has no maximum, but a sum that is not a number: it counts)
      const bool nan = mine > 0 && l_run != l_run;
      const bool any = mine > 0 && (m_used > -INFINITY || nan);
      float m_row = any ? (nan ? fmaxf(m_used, 0.f) : m_used) : -INFINITY, l_row = any ? l_run : 0.f;
      float w_own = any ? 1.f : 0.f, w_other = 0.f;
      bool any_other = false;  // ... and in the second accumulator, once it has been merged
      const int used_rows = tile_tokens * p.tile_heads;
      const bool merge = alt && num > 1;  // with a single key tile the second accumulator has nothing
      // the buffer holds kMergeRows rows: one pass, or two when it is 64 and more rows are in use
      auto merge_chunk = [&](int c4) {  // 16-byte piece c4 of this row in the merge buffer (xor-swizzled against bank conflicts)
        return reinterpret_cast<float4*>(sQ + kTileBytes + ((row % C::kMergeRows) * C::kMergePitch + (c4 ^ (row & 7))) * 16);
      };
      if (merge && wg == 1) {
        for (int pass = 0; pass * C::kMergeRows < used_rows && ok; ++pass) {
          // the first pass needs the previous segment's merge to have been read, the second this one's first pass
          if (!(ok = wait_all(merge_empty, (n_merge & 1) ^ 1))) break;
          ++n_merge;
          if (row / C::kMergeRows == pass && lane_group * 32 < used_rows) {
            sMl[row % C::kMergeRows] = make_float2(m_row, l_row);
#pragma unroll 1
            for (int c = 0; c < D / kOC; ++c) {
              uint32_t v[kOC];
              tmem_ldw(tO + c * kOC, v);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < kOC / 4; ++k)
                *merge_chunk(c * (kOC / 4) + k) = make_float4(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]), __uint_as_float(v[4 * k + 2]),
                                                              __uint_as_float(v[4 * k + 3]));
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(merge_full);
        }
        if (!ok) break;
      } else if (!(alt && wg == 1)) {
        const int item_row = (tok_first + tok) * p.tile_heads + head;  // row of the item: all accumulator tiles
        for (int pass = 0; pass == 0 || (merge && pass * C::kMergeRows < used_rows); ++pass) {
          if (merge) {
            if (!(ok = wait_all(merge_full, n_merge & 1))) break;
            ++n_merge;
          }
          if ((!merge || row / C::kMergeRows == pass) && lane_group * 32 < used_rows) {
            if (merge) {
              const float2 ml = sMl[row % C::kMergeRows];
              const float m = fmaxf(m_row, ml.x);
              w_own = m_row > -INFINITY ? fast_exp2(m_row - m) : 0.f;
              any_other = ml.x > -INFINITY;
              w_other = any_other ? fast_exp2(ml.x - m) : 0.f;
              l_row = l_row * w_own + ml.y * w_other;
              m_row = m;
            }
            const bool direct = g.slot < 0;
            const float inv = direct ? chunk_inverse_sum(l_row) : 1.f;
            const float f0 = w_own * inv, f1 = w_other * inv;
            if (!direct && row_exists) reinterpret_cast<float2*>(p.part_ml)[(size_t)g.slot * p.part_rows + item_row] = make_float2(m_row, l_row);
            // columns c * OC .. of this row, scaled and merged
            auto columns = [&](int c, auto& x) {
              constexpr int OC = sizeof(x) / sizeof(float);
              uint32_t v[OC / kOC][kOC];
#pragma unroll
              for (int h = 0; h < OC / kOC; ++h) tmem_ldw(tO + c * OC + h * kOC, v[h]);
              tmem_wait_ld();
              // (a row whose O counts for nothing may hold anything: no key seen, or no PV run at all)
#pragma unroll
              for (int k = 0; k < OC; ++k) x[k] = any ? __uint_as_float(v[k / kOC][k % kOC]) * f0 : 0.f;
              if (any_other) {
#pragma unroll
                for (int k = 0; k < OC / 4; ++k) {
                  const float4 y = *merge_chunk(c * (OC / 4) + k);
                  x[4 * k] = fmaf(y.x, f1, x[4 * k]);
                  x[4 * k + 1] = fmaf(y.y, f1, x[4 * k + 1]);
                  x[4 * k + 2] = fmaf(y.z, f1, x[4 * k + 2]);
                  x[4 * k + 3] = fmaf(y.w, f1, x[4 * k + 3]);
                }
              }
            };
            // (row numbers count from the item's first output row, or from the slot's first)
            const int to = !row_exists ? -1 : direct ? (tok_first + tok) * p.num_q_heads + head : item_row;
            const size_t first = direct ? (size_t)g.row0 * p.num_q_heads + g.head0 : (size_t)g.slot * p.part_rows;
            if (!direct || p.out_f32)
              chunk_store_rows<D, kOC, 4>(stage, lane, reinterpret_cast<unsigned char*>((direct ? static_cast<float*>(p.out) : p.part_acc) + first * D), to,
                                          columns, [](const float* x) { return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])); });
            else
              chunk_store_rows<D, D % 64 == 0 ? 64 : kOC, 2>(stage, lane, reinterpret_cast<unsigned char*>(static_cast<T*>(p.out) + first * D), to,
                                                             columns, [](const float* x) {
                                                               return make_uint4(Mma16816<T>::pack(x[0], x[1]), Mma16816<T>::pack(x[2], x[3]),
                                                                                 Mma16816<T>::pack(x[4], x[5]), Mma16816<T>::pack(x[6], x[7]));
                                                             });
            if (g.any_bad && row_exists && l_row == l_row)  // (the stores above end with a warp-wide barrier; a row of NaN stays one)
              chunk_add_bad_values<T, D, TPP>(p, g, tok_first + tok, head);
          }
          if (merge) {
            __syncwarp();
            if (lane == 0) mbar_arrive(merge_empty);
          }
        }
        if (!ok) break;
      }
      tc_fence_before();
      if (alt) fence_proxy_async_smem();  // the merge buffer's next user may be a TMA load
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[slot]);
    }
  }

  tc_fence_before();
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the merging kernel may start; it waits for this grid's end)
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---- host side -------------------------------------------------------------------------------
template <typename T, int D, int TPP>
int launch_chunk_typed(const ChunkArgs& a, const ChunkParams& p, int grid, const CUtensorMap& q, const CUtensorMap& v,
                       cudaStream_t stream) {
  constexpr int NQ = chunk_accumulators(D);
  using C = ChunkCfg<D, TPP, NQ>;
  static_assert(C::kTotal <= 227 * 1024, "shared memory exceeds the per-CTA limit");
  auto kern = chunk_tcgen05_kernel<T, D, TPP, NQ>;
  static DeviceOnce configured;  // one per instantiation
  const int rc = configured.run([&] { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal); });
  if (rc != 0) return rc;
  kern<<<grid, C::kThreads, C::kTotal, stream>>>(p, q, v);
  return (int)cudaGetLastError();
}

template <int D, int TPP>
int launch_chunk_shape(const ChunkArgs& a, cudaStream_t stream) {
  ChunkParams p;
  p.k_pool = a.k_pool;
  p.v_pool = a.v_pool;
  p.page_table = a.page_table;
  p.seq_lens = a.seq_lens;
  p.cu_seqlens = a.cu_seqlens;
  p.out = a.out;
  p.status = WaitCtx{static_cast<unsigned int*>(a.status), wait_limit_cycles()};
  p.out_f32 = a.out_f32 ? 1 : 0;
  p.causal = a.causal ? 1 : 0;
  p.window = a.window;
  p.num_seqs = a.num_seqs;
  p.tokens_per_seq = a.cu_seqlens ? 0 : (int)(a.total_tokens / a.num_seqs);
  p.num_q_heads = a.num_q_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.group = a.num_q_heads / a.num_kv_heads;
  const ChunkPlan plan = chunk_plan(a.total_tokens, a.num_q_heads, a.num_kv_heads, D);
  p.tile_heads = plan.tile_heads;
  p.head_blocks = plan.head_blocks;
  p.tile_tokens = plan.tile_tokens;
  p.max_pages_per_seq = a.max_pages_per_seq;
  p.num_pages = a.num_pages;
  p.total_tokens = a.total_tokens;
  p.scale_log2 = a.scale * kLog2e;
  p.part_rows = plan.part_rows;
  p.cuts = reinterpret_cast<ChunkCut*>(a.scratch);
  p.part_ml = reinterpret_cast<float*>(static_cast<unsigned char*>(a.scratch) + plan.ml_offset);
  p.part_acc = reinterpret_cast<float*>(static_cast<unsigned char*>(a.scratch) + plan.acc_offset);

  CUtensorMap mq, mv;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.num_q_heads, (cuuint64_t)a.total_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)a.q_head_stride * 2, (cuuint64_t)a.q_token_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)p.tile_heads, (cuuint32_t)p.tile_tokens};
    if (!encode_map(&mq, a.dtype, 3, a.queries, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return -3;
  }
  if (a.num_pages > 0) {
    const cuuint64_t vdims[3] = {(cuuint64_t)TPP, (cuuint64_t)D, (cuuint64_t)a.num_pages * a.num_kv_heads};
    const cuuint64_t vstrides[2] = {(cuuint64_t)TPP * 2, (cuuint64_t)D * TPP * 2};
    const cuuint32_t vbox[3] = {(cuuint32_t)TPP, (cuuint32_t)D, 1};
    if (!encode_map(&mv, a.dtype, 3, a.v_pool, vdims, vstrides, vbox, TPP == 16 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_64B))
      return -3;
  } else {
    mv = mq;  // never dereferenced: without pages no row sees a key
  }
  const int rc = a.dtype == 0 ? launch_chunk_typed<__half, D, TPP>(a, p, plan.grid, mq, mv, stream)
                              : launch_chunk_typed<__nv_bfloat16, D, TPP>(a, p, plan.grid, mq, mv, stream);
  if (rc != 0) return rc;
  return launch_chunk_merge(a, plan, p.cuts, p.part_ml, p.part_acc, stream);
}

}  // namespace
}  // namespace pal
