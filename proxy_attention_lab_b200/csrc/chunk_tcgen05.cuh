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
//   warp 0      walks the CTA's share, publishes its segments in a ring in shared memory, loads Q and K
//   warp 1      issues every tcgen05.mma and commit
//   warp 2      loads V
//   warps 4..   one softmax warpgroup per accumulator: thread = row = TMEM lane
//
// Operand layouts are those of the prefill kernel (prefill_tcgen05.cuh): Q K-major with the 128-byte swizzle; a key tile
// gathered chunk by chunk from the pages as [D/8][128 tokens][16 B], K-major without swizzle; V pages [D][TPP] K-major with
// the 32- or 64-byte swizzle.  TMEM: S tiles of 128 columns (P overwrites its S tile's first 64; the residual of P, where it
// is fed, the other 64), then O tiles of D columns.  head_dim 256 leaves room for one O tile only: one accumulator with S
// double-buffered.
#pragma once

#include "prefill_tcgen05.cuh"

namespace pal {
namespace {

constexpr int kChunkItemCost = 2;    // fixed cost of an item in key tiles: query load, pipeline fill, epilogue
constexpr int kChunkMinShare = 4;    // smallest share of a CTA, in the same unit
constexpr int kSegRing = 4;

// What one CTA does with one item: key tiles [kt0, kt1) for the rows of the item.
struct ChunkSegment {
  int seq, kv_head;
  int head0, heads;    // first query head of the tile, and how many of its heads exist
  int row0, tokens;    // first query row (token) and how many of the item's tokens exist
  int pos0;            // position of the first token (may be negative)
  int kt0, kt1;
  int key_lo, key_hi;  // keys that some row of the item sees
  int key_cap;         // keys of the sequence
  int alternate;       // one tile of rows: the accumulators take even and odd key tiles
  int slot;            // partial slot to write, -1 = the output itself
  int end;
};

struct ChunkParams {
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

template <int D_, int TPP_, int NQ_>
struct ChunkCfg {
  static constexpr int D = D_, TPP = TPP_, NQ = NQ_, SBUF = NQ == 1 ? 2 : 1;
  using Base = TcCfg<D, TPP, NQ, SBUF>;
  static constexpr int kThreads = 128 + 128 * NQ;
  static constexpr int ST = Base::kStages;
  static constexpr int kQ = 0;
  static constexpr int kK = NQ * Base::kTileBytes;
  static constexpr int kV = kK + ST * Base::kTileBytes;
  static constexpr int kMl = kV + ST * Base::kTileBytes;    // m, l of the second accumulator (alternate segments)
  static constexpr int kBars = kMl + (NQ == 2 ? 1024 : 0);
  static constexpr int kUsed = kBars + 512 + kSegRing * (int)sizeof(ChunkSegment) + 1024;
  static constexpr int kTotal = kUsed < 116 * 1024 ? 116 * 1024 : kUsed;
  // the second Q tile as a buffer of fp32 rows: 16-byte pieces per row (whole groups of eight) and rows that fit
  static constexpr int kMergePitch = (D / 4 + 7) / 8 * 8;
  static constexpr int kMergeRows = Base::kTileBytes / (16 * kMergePitch) < 128 ? 64 : 128;
  static_assert(kMergeRows * kMergePitch * 16 <= Base::kTileBytes, "merge buffer");
};

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

// P = exp2(s * scale - m_ref) of one row, rounded to the input type and packed over the S tile's first 64 columns; the
// rounding residual, where it is fed, over the other 64.  The row sum is taken before the rounding.
template <typename T>
__device__ __forceinline__ void chunk_exp_store(uint32_t tS, const uint32_t (&s)[128], float scale_log2, float m_ref, bool residual, float& l_run) {
  using PK = Mma16816<T>;
  float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  const float2 sc2 = make_float2(scale_log2, scale_log2), nm2 = make_float2(-m_ref, -m_ref);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t hi[32];
    if (PK::kSplitP && residual) {
      uint32_t lo[32];
#pragma unroll
      for (int w = 0; w < 32; ++w) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[64 * h + 2 * w]), __uint_as_float(s[64 * h + 2 * w + 1])), sc2, nm2);
        const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
        hi[w] = PK::pack(e.x, e.y);
        lo[w] = PK::pack_residual(e.x, e.y, hi[w]);
        acc[w & 1] = __fadd2_rn(acc[w & 1], e);
      }
      tmem_st32(tS + 64 + 32 * h, lo);
    } else {
#pragma unroll
      for (int w = 0; w < 32; ++w) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[64 * h + 2 * w]), __uint_as_float(s[64 * h + 2 * w + 1])), sc2, nm2);
        const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
        hi[w] = PK::pack(e.x, e.y);
        acc[w & 1] = __fadd2_rn(acc[w & 1], e);
      }
    }
    tmem_st32(tS + 32 * h, hi);
  }
  l_run += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
}

// bf16 rounds P by up to 2^-9 of its value, which leaves about 0.002 / sqrt(n / 3) per unit of |v| over n keys.  Items with a
// row of fewer than 256 keys, and float32 outputs, get the residual P - bf16(P) through a second set of PV MMAs.
template <typename T>
__device__ __forceinline__ bool chunk_feeds_residual(const ChunkParams& p, const ChunkSegment& g) {
  if (!Mma16816<T>::kSplitP) return false;
  int keys = p.causal ? min(g.pos0 + 1, g.key_cap) : g.key_cap;
  if (p.window > 0) keys = min(keys, p.window);
  return p.out_f32 != 0 || keys < 256;
}

template <typename T, int D, int TPP, int NQ>
__global__ void __launch_bounds__(128 + 128 * NQ, 1)
    chunk_tcgen05_kernel(const __grid_constant__ ChunkParams p, const __grid_constant__ CUtensorMap tm_q,
                         const __grid_constant__ CUtensorMap tm_kpool, const __grid_constant__ CUtensorMap tm_vpool) {
  using C = ChunkCfg<D, TPP, NQ>;
  using B = typename C::Base;
  constexpr int ST = C::ST, SBUF = C::SBUF, kThreadsAll = C::kThreads;
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
  uint64_t* k_full = bars + 2;         // ST
  uint64_t* k_empty = bars + 4;        // ST
  uint64_t* v_full = bars + 6;         // ST
  uint64_t* v_empty = bars + 8;        // ST
  uint64_t* s_full = bars + 10;        // 2: per accumulator, or per S buffer
  uint64_t* p_full = bars + 12;        // 2
  uint64_t* o_done = bars + 14;        // 2: last PV of a segment (NQ = 2), every PV (NQ = 1)
  uint64_t* merge_full = bars + 16;    // 1: the second accumulator's rows are in shared memory
  uint64_t* merge_empty = bars + 17;   // 1
  uint64_t* seg_done = bars + 18;      // 1: the first warpgroup has finished a segment
  uint64_t* seg_full = bars + 20;      // kSegRing
  uint64_t* seg_empty = bars + 24;     // kSegRing
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 30);
  long long* sm_plan = reinterpret_cast<long long*>(bars + 32);  // scan scratch, then the share's first item
  ChunkSegment* segs = reinterpret_cast<ChunkSegment*>(smem + C::kBars + 512);
  static_assert(kSegRing == 4, "barrier layout");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int item_tokens = NQ * p.tile_tokens;
  const int vheads = p.num_kv_heads * p.head_blocks;

  // ---- the CTA's share of the line of items ----
  // thread t sums the cost of a run of sequences; one scan places the runs on the line
  long long share0, share1;
  {
    const int per = (p.num_seqs + kThreadsAll - 1) / kThreadsAll;
    const int sa = min(tid * per, p.num_seqs), sb = min(sa + per, p.num_seqs);
    long long mine = 0;
    for (int s = sa; s < sb; ++s) {
      const ChunkSeq q = chunk_seq(p, s, TPP);
      long long w = 0;
      int lo, hi;
      for (int ta = 0; ta < q.n; ta += item_tokens) w += kChunkItemCost + chunk_keys(p, q, ta, min(ta + item_tokens, q.n), lo, hi);
      mine += w * vheads;
    }
    long long inc = mine;
#pragma unroll
    for (int sh = 1; sh < 32; sh <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, sh);
      if (lane >= sh) inc += up;
    }
    if (lane == 31) sm_plan[warp] = inc;
    if (tid == 0) {
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&k_full[i], 1);
        mbar_init(&k_empty[i], 1);
        mbar_init(&v_full[i], 1);
        mbar_init(&v_empty[i], 1);
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 4);
        mbar_init(&o_done[i], 1);
      }
      mbar_init(merge_full, 4);
      mbar_init(merge_empty, 4);
      mbar_init(seg_done, 4);
      for (int i = 0; i < kSegRing; ++i) {
        mbar_init(&seg_full[i], 1);
        mbar_init(&seg_empty[i], 2 + 4 * NQ);
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
    }
    long long share = (total + gridDim.x - 1) / gridDim.x;
    if (share < kChunkMinShare) share = kChunkMinShare;
    share0 = min(share * blockIdx.x, total);
    share1 = min(share0 + share, total);
    __syncthreads();
    const long long start = before + inc - mine;
    if (share0 < share1 && share0 >= start && share0 < start + mine) {
      // the share begins in this thread's run: find the item
      long long at = start;
      int s = sa, vh = 0, ta = 0;
      for (; s < sb; ++s) {
        const ChunkSeq q = chunk_seq(p, s, TPP);
        long long w = 0;
        int lo, hi;
        for (int t = 0; t < q.n; t += item_tokens) w += kChunkItemCost + chunk_keys(p, q, t, min(t + item_tokens, q.n), lo, hi);
        if (share0 < at + w * vheads) {
          vh = (int)((share0 - at) / w);
          at += vh * w;
          for (;; ta += item_tokens) {
            const int c = kChunkItemCost + chunk_keys(p, q, ta, min(ta + item_tokens, q.n), lo, hi);
            if (share0 < at + c) break;
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
    // =============================== segments, Q and K ===============================
    if (share0 >= share1) {
      if (lane == 0) p.cuts[blockIdx.x].parts = 0;
    }
    int s = 0, vh = 0, ta = 0;
    long long at = share0, share = 1;
    if (share0 < share1) {
      s = (int)sm_plan[0];
      vh = (int)sm_plan[1];
      ta = (int)sm_plan[2];
      at = sm_plan[3];
      share = sm_plan[4];
    }
    __syncwarp();
    ChunkSeq q = share0 < share1 ? chunk_seq(p, s, TPP) : ChunkSeq{};
    uint32_t n_seg = 0, n_tile = 0;  // segments and key tiles so far (ring positions)
    bool prev_alternate = false;
    bool cut_written = false;
    int ok = 1;
    while (ok) {
      // ---- next segment of the share (the same computation on every lane) ----
      ChunkSegment g;
      g.end = 1;
      while (at < share1) {
        const int tb = min(ta + item_tokens, q.n);
        int lo = 0, hi = 0, nt = 0, cost = 0;
        if (q.n > 0) {
          nt = chunk_keys(p, q, ta, tb, lo, hi);
          cost = kChunkItemCost + nt;
          const long long first = at + kChunkItemCost;  // place of key tile 0 on the line
          const int t0 = (int)min((long long)nt, max(0LL, share0 - first)), t1 = (int)max(0LL, min((long long)nt, share1 - first));
          if (t1 > t0 || (nt == 0 && at >= share0)) {
            g.end = 0;
            g.seq = s;
            g.kv_head = vh / p.head_blocks;
            const int hb = vh - g.kv_head * p.head_blocks;
            g.head0 = g.kv_head * p.group + hb * p.tile_heads;
            g.heads = min(p.tile_heads, p.group - hb * p.tile_heads);
            g.row0 = q.row0 + ta;
            g.tokens = tb - ta;
            g.pos0 = q.len - q.n + ta;
            g.kt0 = lo / kTile + t0;
            g.kt1 = lo / kTile + t1;
            g.key_lo = lo;
            g.key_hi = hi;
            g.key_cap = q.cap;
            g.alternate = NQ == 2 && g.tokens <= p.tile_tokens;
            g.slot = t0 > 0 ? 2 * (int)blockIdx.x : (t1 < nt ? 2 * (int)blockIdx.x + 1 : -1);
            if (t0 == 0 && t1 < nt && lane == 0) {
              // this CTA holds the item's first part: tell the merging kernel where the others are
              ChunkCut c;
              c.parts = (int)((first + nt - 1) / share) - (int)blockIdx.x + 1;
              c.row0 = g.row0;
              c.tokens = g.tokens;
              c.head0 = g.head0;
              c.heads = g.heads;
              p.cuts[blockIdx.x] = c;
              cut_written = true;
            }
          }
        }
        // advance: row tiles, then heads, then sequences
        at += cost;
        ta += item_tokens;
        if (ta >= q.n) {
          ta = 0;
          if (q.n <= 0 || ++vh == vheads) {
            vh = 0;
            ++s;
            if (at < share1) q = chunk_seq(p, s, TPP);
          }
        }
        if (!g.end) break;
      }
      // ---- publish it ----
      const int slot = n_seg % kSegRing;
      if (lane == 0) {
        ok = mbar_wait(&seg_empty[slot], ((n_seg / kSegRing) & 1) ^ 1, p.status);
        if (ok) {
          segs[slot] = g;
          mbar_arrive(&seg_full[slot]);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok || g.end) break;
      if (g.kt0 < g.kt1) {
        // ---- Q: free once the last QK^T of the previous segment with keys has run; the second tile also serves as the
        // merge buffer of alternate segments ----
        if (lane == 0) {
          ok = mbar_wait(q_empty, (n_seg & 1) ^ 1, p.status);
          if (ok && !g.alternate && prev_alternate) ok = mbar_wait(seg_done, (n_seg & 1) ^ 1, p.status);
          if (ok) {
            const int tiles = NQ == 2 && !g.alternate ? 2 : 1;
            mbar_arrive_expect_tx(q_full, tiles * kBlocks * p.tile_heads * p.tile_tokens * 128);
            for (int t = 0; t < tiles; ++t)
              for (int kb = 0; kb < kBlocks; ++kb)
                tma_load_3d(sQ + t * kTileBytes + kb * kBlockBytes, &tm_q, kb * 64, g.head0, g.row0 + t * p.tile_tokens, q_full);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
      } else if (lane == 0) {
        // no keys: the segment passes through the barriers that count segments
        ok = mbar_wait(q_empty, (n_seg & 1) ^ 1, p.status);
        if (ok) mbar_arrive(q_full);
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      prev_alternate = g.alternate != 0;
      ++n_seg;
      // ---- K ----
      const uint32_t* pages = p.page_table + (size_t)g.seq * p.max_pages_per_seq;
      for (int j = g.kt0; j < g.kt1 && ok; ++j, ++n_tile) {
        const int st = n_tile % ST;
        // pages [pg0, pg1) of the tile hold visible keys; the others are not fetched (their columns of S are masked)
        const int pg0 = max(0, g.key_lo - j * kTile) / TPP;
        const int pg1 = (min(kTile, g.key_hi - j * kTile) + TPP - 1) / TPP;
        uint32_t pid = 0;
        if (lane < kPagesPerTile) {
          pid = pages[j * kPagesPerTile + min(max(lane, pg0), pg1 - 1)];
          if ((long long)pid >= p.num_pages) pid = (uint32_t)(p.num_pages - 1);
        }
        if (lane == 0) ok = mbar_wait(&k_empty[st], ((n_tile / ST) & 1) ^ 1, p.status);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        constexpr int kChunks = D / 8, kGroups = kPagesPerTile / 4;
        constexpr int kGroupBytes = 4 * TPP * 16;
        const int g0 = pg0 >> 2, g1 = (pg1 + 3) >> 2;
        if (lane == 0) mbar_arrive_expect_tx(&k_full[st], kChunks * (g1 - g0) * kGroupBytes);
        __syncwarp();
#pragma unroll
        for (int op0 = 0; op0 < kChunks * kGroups; op0 += 32) {
          const int op = op0 + lane;
          const int c = op / kGroups, gr = op % kGroups;
          int rows[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) rows[i] = ((int)__shfl_sync(0xffffffffu, pid, (4 * gr + i) & 31) * p.num_kv_heads + g.kv_head) * kChunks + c;
          if (op < kChunks * kGroups && gr >= g0 && gr < g1)
            tma_gather4(sK + st * kTileBytes + c * B::kChunkBytes + gr * kGroupBytes, &tm_kpool, 0, rows[0], rows[1], rows[2], rows[3],
                        &k_full[st]);
        }
      }
    }
    if (lane == 0 && share0 < share1 && !cut_written) p.cuts[blockIdx.x].parts = 0;
  } else if (warp == 1) {
    // =============================== MMA issuer ===============================
    constexpr int F = Fmt<T>::kCode;
    constexpr uint32_t idesc_qk = make_idesc(128, F, F, 0);
    constexpr uint32_t idesc_pv = make_idesc(D, F, F, 0);
    const uint64_t q_desc = make_desc(smem_u32(sQ), 16, 1024, kLayoutSw128);
    const uint64_t k_desc = make_desc(smem_u32(sK), B::kChunkBytes, 128, kLayoutNone);
    const uint64_t v_desc = make_desc(smem_u32(sV), 16, 8 * TPP * 2, TPP == 16 ? kLayoutSw32 : kLayoutSw64);
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)) != 0; };
    uint32_t n_seg = 0, kt = 0, vt = 0;  // segments, key tiles whose QK^T / PV have been issued
    uint32_t n_p0 = 0, n_p1 = 0;         // P tiles taken from each accumulator (NQ = 2)
    bool ok = true;
    // S(si) = Q(tile) . K^T of the next key tile
    auto issue_qk = [&](int q_tile, int si, int st) {
      if (!elect_one()) return;
      const uint32_t d_tmem = tmem_base + si * kTile;
      const uint64_t qa = q_desc + (uint64_t)(q_tile * (kTileBytes >> 4)), kb = k_desc + (uint64_t)(st * (kTileBytes >> 4));
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        tc_mma_ss(d_tmem, qa + (uint64_t)(((ks >> 2) * kBlockBytes + (ks & 3) * 32) >> 4), kb + (uint64_t)((ks * 2 * B::kChunkBytes) >> 4), idesc_qk,
                  ks > 0);
      tc_commit(&s_full[si]);
    };
    // O(acc) += P(si) . V over the 16-key steps [kk0, kk1); `first`: the accumulator starts afresh
    auto issue_pv = [&](int acc, int si, int st, int kk0, int kk1, bool first, bool residual) {
      if (!elect_one()) return;
      const uint32_t d_tmem = tmem_base + B::kOBase + acc * B::DP;
      const uint64_t vb = v_desc + (uint64_t)(st * (kTileBytes >> 4));
      uint32_t accumulate = first ? 0u : 1u;
      for (int part = 0; part < (residual ? 2 : 1); ++part) {
        const uint32_t a_tmem = tmem_base + si * kTile + part * 64;
        if (kk0 == 0 && kk1 == kTile / 16) {
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk) {
            const int off = TPP == 16 ? kk * kPageBytes : (kk >> 1) * kPageBytes + (kk & 1) * 32;
            tc_mma_ts(d_tmem, a_tmem + kk * 8, vb + (uint64_t)(off >> 4), idesc_pv, accumulate);
            accumulate = 1u;
          }
        } else {
#pragma unroll 1
          for (int kk = kk0; kk < kk1; ++kk) {
            const int off = TPP == 16 ? kk * kPageBytes : (kk >> 1) * kPageBytes + (kk & 1) * 32;
            tc_mma_ts(d_tmem, a_tmem + kk * 8, vb + (uint64_t)(off >> 4), idesc_pv, accumulate);
            accumulate = 1u;
          }
        }
      }
    };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) tc_commit(bar);
    };
    while (ok) {
      const int slot = n_seg % kSegRing;
      ok = wait_all(&seg_full[slot], (n_seg / kSegRing) & 1);
      if (!ok) break;
      const ChunkSegment g = segs[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[slot]);
      if (g.end) break;
      ok = wait_all(q_full, n_seg & 1);
      ++n_seg;
      if (!ok) break;
      if (g.kt0 >= g.kt1) {
        if (lane == 0) mbar_arrive(q_empty);
        continue;
      }
      const bool residual = chunk_feeds_residual<T>(p, g);
      const int num = g.kt1 - g.kt0;
      auto steps = [&](int j, int& kk0, int& kk1) {
        kk0 = max(0, g.key_lo - j * kTile) >> 4;
        kk1 = (min(kTile, g.key_hi - j * kTile) + 15) >> 4;
      };
      auto wait_k = [&]() {
        const bool r = wait_all(&k_full[kt % ST], (kt / ST) & 1);
        tc_fence_after();
        return r;
      };
      auto wait_v = [&]() { return wait_all(&v_full[vt % ST], (vt / ST) & 1); };
      auto wait_p = [&](int si) {
        const uint32_t n = NQ == 1 ? vt >> 1 : (si ? n_p1++ : n_p0++);  // (the two S buffers of one accumulator take turns)
        const bool r = wait_all(&p_full[si], n & 1);
        tc_fence_after();
        return r;
      };
      int kk0, kk1;
      if (NQ == 1) {
        // one accumulator, two S buffers: QK^T of tile i + 1 runs under the softmax of tile i
        ok = wait_k();
        if (!ok) break;
        issue_qk(0, kt & 1, kt % ST);
        commit(&k_empty[kt % ST]);
        ++kt;
        if (num == 1) commit(q_empty);
        for (int i = 0; i < num && ok; ++i) {
          if (i + 1 < num) {
            ok = wait_k();
            if (!ok) break;
            issue_qk(0, kt & 1, kt % ST);
            commit(&k_empty[kt % ST]);
            ++kt;
            if (i + 2 == num) commit(q_empty);
          }
          const int si = vt & 1;
          ok = wait_v() && wait_p(si);
          if (!ok) break;
          steps(g.kt0 + i, kk0, kk1);
          issue_pv(0, si, vt % ST, kk0, kk1, i == 0, residual);
          commit(&o_done[si]);
          commit(&v_empty[vt % ST]);
          ++vt;
        }
      } else if (g.alternate) {
        for (int i = 0; i < 2 && i < num && ok; ++i) {
          ok = wait_k();
          if (!ok) break;
          issue_qk(0, i, kt % ST);
          commit(&k_empty[kt % ST]);
          ++kt;
        }
        if (ok && num <= 2) commit(q_empty);
        for (int i = 0; i < num && ok; ++i) {
          const int a = i & 1;
          ok = wait_v() && wait_p(a);
          if (!ok) break;
          steps(g.kt0 + i, kk0, kk1);
          issue_pv(a, a, vt % ST, kk0, kk1, i < 2, residual);
          commit(&v_empty[vt % ST]);
          ++vt;
          if (i + 2 < num) {
            ok = wait_k();
            if (!ok) break;
            issue_qk(0, a, kt % ST);
            commit(&k_empty[kt % ST]);
            ++kt;
            if (i + 3 == num) commit(q_empty);
          } else {
            commit(&o_done[a]);
          }
        }
      } else {
        ok = wait_k();
        if (!ok) break;
        issue_qk(0, 0, kt % ST);
        issue_qk(1, 1, kt % ST);
        commit(&k_empty[kt % ST]);
        ++kt;
        if (num == 1) commit(q_empty);
        for (int i = 0; i < num && ok; ++i) {
          ok = wait_v();
          steps(g.kt0 + i, kk0, kk1);
          for (int a = 0; a < 2 && ok; ++a) {
            ok = wait_p(a);
            if (!ok) break;
            issue_pv(a, a, vt % ST, kk0, kk1, i == 0, residual);
            if (i + 1 < num) {
              if (a == 0) ok = wait_k();
              if (!ok) break;
              issue_qk(a, a, kt % ST);
            } else {
              commit(&o_done[a]);
            }
          }
          if (!ok) break;
          commit(&v_empty[vt % ST]);
          ++vt;
          if (i + 1 < num) {
            commit(&k_empty[kt % ST]);
            ++kt;
            if (i + 2 == num) commit(q_empty);
          }
        }
      }
      __syncwarp();
    }
  } else if (warp == 2) {
    // =============================== V ===============================
    uint32_t n_seg = 0, n_tile = 0;
    int ok = 1;
    while (ok) {
      const int slot = n_seg % kSegRing;
      ok = __all_sync(0xffffffffu, mbar_wait(&seg_full[slot], (n_seg / kSegRing) & 1, p.status));
      if (!ok) break;
      const ChunkSegment g = segs[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[slot]);
      if (g.end) break;
      ++n_seg;
      const uint32_t* pages = p.page_table + (size_t)g.seq * p.max_pages_per_seq;
      for (int j = g.kt0; j < g.kt1 && ok; ++j, ++n_tile) {
        const int st = n_tile % ST;
        const int pg0 = max(0, g.key_lo - j * kTile) / TPP;
        const int pg1 = (min(kTile, g.key_hi - j * kTile) + TPP - 1) / TPP;
        uint32_t pid = 0;
        if (lane >= pg0 && lane < pg1) {
          pid = pages[j * kPagesPerTile + lane];
          if ((long long)pid >= p.num_pages) pid = (uint32_t)(p.num_pages - 1);
        }
        if (lane == 0) {
          ok = mbar_wait(&v_empty[st], ((n_tile / ST) & 1) ^ 1, p.status);
          if (ok) mbar_arrive_expect_tx(&v_full[st], (pg1 - pg0) * kPageBytes);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        if (lane >= pg0 && lane < pg1)
          tma_load_3d(sV + st * kTileBytes + lane * kPageBytes, &tm_vpool, 0, 0, (int)(pid * p.num_kv_heads + g.kv_head), &v_full[st]);
      }
    }
  }
  } else {
    if (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // =============================== softmax warpgroups ===============================
    const int wg = (warp - 4) >> 2;
    const int lane_group = warp & 3;
    const int row = lane_group * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(lane_group * 32) << 16;
    const uint32_t tO = tmem_base + lane_addr + B::kOBase + wg * B::DP;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)) != 0; };
    // Phases: with one S buffer the s_full of this accumulator has completed n_s times and its o_done n_o times; with two
    // buffers, taken in turns, both follow from the number of key tiles n_v.
    uint32_t n_seg = 0, n_s = 0, n_o = 0, n_v = 0, n_merge = 0;
    bool ok = true;
    while (ok) {
      const int slot = n_seg % kSegRing;
      ok = wait_all(&seg_full[slot], (n_seg / kSegRing) & 1);
      if (!ok) break;
      const ChunkSegment g = segs[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[slot]);
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
      // ... and the narrowest range over the tile's tokens: key tiles inside it need no mask
      const int pos_a = g.pos0 + tok_first, pos_b = pos_a + p.tile_tokens - 1;
      const int all_hi = p.causal ? min(pos_a, g.key_cap - 1) : g.key_cap - 1;
      const int all_lo = p.window > 0 && pos_b >= p.window ? pos_b - p.window + 1 : 0;
      const bool residual = chunk_feeds_residual<T>(p, g);
      float m_used = -INFINITY, l_run = 0.f;
      const int num = g.kt1 - g.kt0;
      int mine = 0;  // key tiles this accumulator has taken
      for (int i = 0; i < num; ++i) {
        if (alt && (i & 1) != wg) {
          ++n_v;
          continue;
        }
        const int j = g.kt0 + i;
        const int si = SBUF == 2 ? (int)(n_v & 1) : wg;
        const uint32_t tS = tmem_base + lane_addr + si * kTile;
        if (!(ok = wait_all(&s_full[si], (SBUF == 2 ? n_v >> 1 : n_s) & 1))) break;
        ++n_s;
        tc_fence_after();
        if (warp_works) {
          uint32_t sc[128];
          tmem_ld128(tS, sc);
          tmem_wait_ld();
          const bool need_mask = (j + 1) * kTile - 1 > all_hi || j * kTile < all_lo;
          if (need_mask) {
            const int rh = hi - j * kTile, rl = lo - j * kTile;
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (c > rh || c < rl) sc[c] = 0xff800000u;
          }
          const float mx = row_max128(sc) * p.scale_log2;  // scale > 0: the maximum commutes with the scaling
          const float m_new = fmaxf(m_used, mx);
          if (mine == 0) {
            m_used = m_new;
          } else if (__any_sync(0xffffffffu, m_new > m_used + kRescaleThreshold)) {
            // O must be stable.  With one S buffer per accumulator QK^T of this tile was issued after PV of the previous
            // one, so it is; with two, that PV may still run.
            if (SBUF == 2) {
              if (!(ok = wait_all(&o_done[(n_v - 1) & 1], ((n_v - 1) >> 1) & 1))) break;
              tc_fence_after();
            }
            const float f = m_new > m_used ? fast_exp2(m_used - m_new) : 1.f;
#pragma unroll
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
          const float m_ref = m_used > -INFINITY ? m_used : 0.f;
          chunk_exp_store<T>(tS, sc, p.scale_log2, m_ref, residual, l_run);
          tmem_wait_st();
        }
        ++mine;
        // V rows of slots that no row of the item sees (past the last key, before the window, never written) would be
        // multiplied by P = 0, which is not 0 if they hold an infinity or a NaN: zero them in the 16-key steps that are used.
        if (wg == 0 || alt) {
          const int c_lo = max(0, g.key_lo - j * kTile), c_hi = min(kTile, g.key_hi - j * kTile);
          if ((c_lo | c_hi) & 15) {
            const int st = (int)(n_v % ST);
            if (!(ok = wait_all(&v_full[st], (n_v / ST) & 1))) break;
            unsigned char* vt = sV + st * kTileBytes;
            for (int dr = row; dr < D; dr += 128) {
              const int sw = TPP == 16 ? ((dr >> 2) & 1) : ((dr >> 1) & 3);
              auto clear = [&](int from, int to) {
                for (int c = from; c < to; ++c) {
                  const int s = c % TPP;
                  *reinterpret_cast<uint16_t*>(vt + (c / TPP) * kPageBytes + dr * (TPP * 2) + ((((s >> 3) ^ sw) << 4) | ((s & 7) << 1))) = 0;
                }
              };
              clear(c_lo & ~15, c_lo);
              clear(c_hi, (c_hi + 15) & ~15);
            }
            fence_proxy_async_smem();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[si]);
        ++n_v;
      }
      if (!ok) break;
      // ---- epilogue ----
      // O is complete (its last PV committed): NQ = 2 commits once per segment and accumulator that had key tiles
      if (mine > 0) {
        if (SBUF == 2) {
          ok = wait_all(&o_done[(n_v - 1) & 1], ((n_v - 1) >> 1) & 1);
        } else {
          ok = wait_all(&o_done[wg], n_o & 1);
          ++n_o;
        }
        if (!ok) break;
        tc_fence_after();
      }
      const bool any = mine > 0 && m_used > -INFINITY;
      float m_row = any ? m_used : -INFINITY, l_row = any ? l_run : 0.f;
      float w_own = any ? 1.f : 0.f, w_other = 0.f;
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
            sMl[row] = make_float2(m_row, l_row);
#pragma unroll
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
        const long long tok_row = (long long)g.row0 + tok_first + tok;
        const size_t out_row = (size_t)tok_row * p.num_q_heads + g.head0 + head;
        const int item_row = (tok_first + tok) * p.tile_heads + head;  // row of the item: all accumulator tiles
        for (int pass = 0; pass == 0 || (merge && pass * C::kMergeRows < used_rows); ++pass) {
          if (merge) {
            if (!(ok = wait_all(merge_full, n_merge & 1))) break;
            ++n_merge;
          }
          if ((!merge || row / C::kMergeRows == pass) && lane_group * 32 < used_rows) {
            if (merge) {
              const float2 ml = sMl[row];
              const float m = fmaxf(m_row, ml.x);
              w_own = m_row > -INFINITY ? fast_exp2(m_row - m) : 0.f;
              w_other = ml.x > -INFINITY ? fast_exp2(ml.x - m) : 0.f;
              l_row = l_row * w_own + ml.y * w_other;
              m_row = m;
            }
            const bool direct = g.slot < 0;
            const float inv = direct ? (l_row > 0.f ? 1.f / l_row : (l_row == 0.f ? 0.f : l_row)) : 1.f;
            const float f0 = w_own * inv, f1 = w_other * inv;
            if (!direct && row_exists) reinterpret_cast<float2*>(p.part_ml)[(size_t)g.slot * p.part_rows + item_row] = make_float2(m_row, l_row);
#pragma unroll
            for (int c = 0; c < D / kOC; ++c) {
              float x[kOC];
              if (mine > 0) {
                uint32_t v[kOC];
                tmem_ldw(tO + c * kOC, v);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < kOC; ++k) x[k] = f0 != 0.f ? __uint_as_float(v[k]) * f0 : 0.f;
              } else {
#pragma unroll
                for (int k = 0; k < kOC; ++k) x[k] = 0.f;
              }
              if (merge && f1 != 0.f) {
#pragma unroll
                for (int k = 0; k < kOC / 4; ++k) {
                  const float4 y = *merge_chunk(c * (kOC / 4) + k);
                  x[4 * k] = fmaf(y.x, f1, x[4 * k]);
                  x[4 * k + 1] = fmaf(y.y, f1, x[4 * k + 1]);
                  x[4 * k + 2] = fmaf(y.z, f1, x[4 * k + 2]);
                  x[4 * k + 3] = fmaf(y.w, f1, x[4 * k + 3]);
                }
              }
              if (!row_exists) continue;
              if (!direct || p.out_f32) {
                float4* dst = reinterpret_cast<float4*>(direct ? static_cast<float*>(p.out) + out_row * D
                                                               : p.part_acc + ((size_t)g.slot * p.part_rows + item_row) * D) +
                              c * (kOC / 4);
#pragma unroll
                for (int k = 0; k < kOC / 4; ++k) dst[k] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
              } else {
                uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_row * D) + c * (kOC / 8);
#pragma unroll
                for (int k = 0; k < kOC / 8; ++k)
                  dst[k] = make_uint4(Mma16816<T>::pack(x[8 * k], x[8 * k + 1]), Mma16816<T>::pack(x[8 * k + 2], x[8 * k + 3]),
                                      Mma16816<T>::pack(x[8 * k + 4], x[8 * k + 5]), Mma16816<T>::pack(x[8 * k + 6], x[8 * k + 7]));
              }
            }
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
      if (wg == 0 && lane == 0) mbar_arrive(seg_done);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---- host side -------------------------------------------------------------------------------
template <typename T, int D, int TPP>
int launch_chunk_typed(const ChunkArgs& a, const ChunkParams& p, int grid, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                       cudaStream_t stream) {
  constexpr int NQ = chunk_accumulators(D);
  using C = ChunkCfg<D, TPP, NQ>;
  static_assert(C::kTotal <= 227 * 1024, "shared memory exceeds the per-CTA limit");
  auto kern = chunk_tcgen05_kernel<T, D, TPP, NQ>;
  static DeviceOnce configured;  // one per instantiation
  const int rc = configured.run([&] { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal); });
  if (rc != 0) return rc;
  kern<<<grid, C::kThreads, C::kTotal, stream>>>(p, q, k, v);
  return (int)cudaGetLastError();
}

template <int D, int TPP>
int launch_chunk_shape(const ChunkArgs& a, cudaStream_t stream) {
  ChunkParams p;
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

  CUtensorMap mq, mk, mv;
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
    const cuuint64_t kdims[2] = {(cuuint64_t)TPP * 8, (cuuint64_t)a.num_pages * a.num_kv_heads * (D / 8)};
    const cuuint64_t kstrides[1] = {(cuuint64_t)TPP * 16};
    const cuuint32_t kbox[2] = {(cuuint32_t)TPP * 8, 1};
    if (!encode_map(&mk, a.dtype, 2, a.k_pool, kdims, kstrides, kbox, CU_TENSOR_MAP_SWIZZLE_NONE)) return -3;
  } else {
    mk = mv = mq;  // never dereferenced: without pages no row sees a key
  }
  const int rc = a.dtype == 0 ? launch_chunk_typed<__half, D, TPP>(a, p, plan.grid, mq, mk, mv, stream)
                              : launch_chunk_typed<__nv_bfloat16, D, TPP>(a, p, plan.grid, mq, mk, mv, stream);
  if (rc != 0) return rc;
  return launch_chunk_merge(a, plan, p.cuts, p.part_ml, p.part_acc, stream);
}

}  // namespace
}  // namespace pal
