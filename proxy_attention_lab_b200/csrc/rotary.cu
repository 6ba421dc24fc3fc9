// Rotary position embedding for sm_100a: the rotation of queries / keys by one to four position axes, alone
// (rotary_embedding) or on the way into the page pools (fill_kv_pages_rotary).
//
// Mathematics.  Frequency i (of R / 2) turns one pair of elements (a, b) of every head by the angle
// t = position[axis(i)] * inv_freq[i]:   a' = m (a cos t - b sin t),   b' = m (b cos t + a sin t),
// with (a, b) = elements (i, i + R/2) or (2i, 2i + 1), and m a common magnitude.  Elements past R pass through.
// The angle of a far position is large (position 10^6 times frequency 1), and its fp32 product would be off by up to
// 2^-24 * 10^6 = 0.06 rad, so product and reduction to a fraction of a turn are taken in fp64 (exact product for
// positions below 2^29; above, product and factor are off by 3e-16 of the angle, 1e-7 turns at 2^31); the fraction, at most half a
// turn, is then good to 2^-25 turns in fp32 and sincospif does the rest.
//
// Bound: memory.  A rotated element costs 4 bytes of traffic and ~3 flops; the angle, ~60 instructions, is shared by all
// heads of a token.  So a block takes a few tokens, computes their sines and cosines once into shared memory, and then a
// thread owns one unit - 2 V elements of a head row, V frequencies - of one token, takes its angles into registers and walks
// over the heads with 16-byte loads and stores (V = 8).  Few tokens: one per block, and the heads spread over all threads;
// many: sixteen per block.
//
// fill_kv_pages_rotary is one launch of blocks in two roles: rotate queries and keys, and move the values into the V pool.
//   K pool [P, Hkv, D/8, TPP, 8]: a unit is whole 16-byte chunks; a warp reads 128 contiguous bytes of a row and writes runs
//     of a few tokens' neighbouring 16-byte chunks.
//   V pool [P, Hkv, D, TPP]: eight consecutive slots of a page are 16 contiguous bytes of a head-dim row.  A block stages 64
//     tokens (and the 7 that follow them) of one head in shared memory and finds the octets: runs of eight tokens that fill
//     an aligned group of eight slots.  An octet belongs to the block that holds its first token, hence the halo: prompts
//     start anywhere in a page, and cutting octets at block borders would turn a fifth of the stores into 2-byte ones.
//     ldmatrix.trans does the transposition: its row addresses are free, so row 2 t + b of matrix k is given the address of
//     token 2 k + b of octet t, and each lane receives the eight tokens of one head-dim element of octet t in four
//     registers - one 16-byte store.  The rest (single tokens, ends of runs) leaves in 2-byte stores.
#include "append.cuh"
#include "common.cuh"
#include "launch.h"

namespace pal {
namespace {

constexpr int kThreads = 256;
constexpr int kTokensPerTile = 64;               // list tokens a V block owns (8 where that leaves SMs idle)
constexpr int kTileTokens = kTokensPerTile + 7;  // ... and stages: the octet that starts at its last token ends 7 later
constexpr int kTokensPerBlock = 16;              // of a rotating block, when there are enough tokens to fill the GPU
// Bytes of a rotating block's table of angles.  A launch has 48 KB in all without asking for more, of which the lists of a V block
// take 1152 bytes (they are static, so every block has them).
constexpr size_t kTableBytes = 46 * 1024;

struct RotaryParams {
  RotationArgs rot;
  RowsView src_q, src_k, src_v;
  void* q_out;
  long long q_out_token_stride, q_out_head_stride;
  FillArgs fill;
  int hq;               // query heads to rotate (0 = none)
  int block_tokens;     // tokens of a rotating block
  int head_splits;      // rotating blocks that share a group of tokens: each takes a range of heads
  unsigned v_blocks;
  int v_tokens;         // tokens a V block owns
  int v_vec;            // new_values can be read in 16-byte vectors
};

template <int V>
struct Vec;
template <>
struct Vec<8> { using type = uint4; };
template <>
struct Vec<4> { using type = uint2; };
template <>
struct Vec<1> { using type = uint16_t; };

template <typename T, int V>
union Elems {
  typename Vec<V>::type v;
  T e[V];
  __device__ Elems() {}
};

// Which axis frequency i belongs to.  Blocked: the first sections[0] frequencies are axis 0's, and so on.  Interleaved:
// frequencies go round the axes, and axis a > 0 stops after its sections[a] (those that are left over are axis 0's).
__device__ __forceinline__ int axis_of(const RotationArgs& r, int i) {
  if (r.num_axes <= 1) return 0;
  if (r.section_order == 0) {
    int a = 0, end = r.sections[0];
    while (a + 1 < r.num_axes && i >= end) end += r.sections[++a];
    return a;
  }
  const int a = i % r.num_axes;
  return i / r.num_axes < r.sections[a] ? a : 0;
}

// Cosine and sine, times the magnitude, of frequency i at a token's position.
__device__ __forceinline__ float2 cos_sin(const RotationArgs& r, long long token, int i) {
  const long long at = axis_of(r, i) * r.positions_axis_stride + token;
  const double pos = r.positions_64bit ? (double)static_cast<const long long*>(r.positions)[at] : (double)static_cast<const int*>(r.positions)[at];
  double turns = pos * (double)r.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
  turns -= rint(turns);
  float sn, cs;
  sincospif(2.0f * (float)turns, &sn, &cs);
  return make_float2(cs * r.magnitude, sn * r.magnitude);
}

template <int V>
struct Angles {
  float c[V], s[V];
};

// Unit u of a head row: two vectors of V elements at `first` and `second`; units past the rotated elements pass through
// (their second vector may lie past the row: second < 0).
template <int V, bool ADJACENT>
struct Unit {
  int first, second;
  bool turns;
  __device__ __forceinline__ Unit(int u, int half, int head_dim) {
    const int rotated = half / V;
    turns = u < rotated;
    if (turns) {
      first = ADJACENT ? 2 * V * u : V * u;
      second = ADJACENT ? first + V : half + V * u;
    } else {
      first = 2 * half + 2 * V * (u - rotated);
      second = first + V < head_dim ? first + V : -1;
    }
  }
};

template <typename T, int V, bool ADJACENT>
__device__ __forceinline__ void turn(Elems<T, V>& a, Elems<T, V>& b, const Angles<V>& g) {
  using M = Mma16816<T>;
  if (ADJACENT && V == 1) {
    const float x = M::to_float(a.e[0]), y = M::to_float(b.e[0]);
    a.e[0] = M::from_float(x * g.c[0] - y * g.s[0]);
    b.e[0] = M::from_float(y * g.c[0] + x * g.s[0]);
  } else if (ADJACENT) {
    // vector a holds pairs 0 .. V/2 - 1, vector b the others
#pragma unroll
    for (int e = 0; e < V; ++e) {
      Elems<T, V>& w = e < V / 2 ? a : b;
      const int k = 2 * (e % (V / 2 > 0 ? V / 2 : 1));
      const float x = M::to_float(w.e[k]), y = M::to_float(w.e[k + 1 < V ? k + 1 : k]);
      w.e[k] = M::from_float(x * g.c[e] - y * g.s[e]);
      w.e[k + 1 < V ? k + 1 : k] = M::from_float(y * g.c[e] + x * g.s[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float x = M::to_float(a.e[e]), y = M::to_float(b.e[e]);
      a.e[e] = M::from_float(x * g.c[e] - y * g.s[e]);
      b.e[e] = M::from_float(y * g.c[e] + x * g.s[e]);
    }
  }
}

// (page, slot) of token t, or page = -1 when the token has to be skipped
__device__ __forceinline__ void destination(const FillArgs& f, long long t, long long& page, int& slot) {
  const uint32_t *table = static_cast<const uint32_t*>(f.page_table), *map = static_cast<const uint32_t*>(f.query_to_seq_map);
  if (f.slot_mapping)
    token_destination<true>(t, f.slot_mapping, table, f.write_positions, map, f.num_seqs, f.tokens_per_page, f.num_pages, f.max_pages_per_seq, page, slot);
  else
    token_destination<false>(t, f.slot_mapping, table, f.write_positions, map, f.num_seqs, f.tokens_per_page, f.num_pages, f.max_pages_per_seq, page, slot);
}

// A rotating block: tokens [t0, t0 + block_tokens) of heads [head0, head1), counting the queries' heads first and then the
// keys'.  `table`: [token][2][num_freqs] cosines and sines.
template <typename T, int V, bool ADJACENT>
__device__ __forceinline__ void rotate(const RotaryParams& p, unsigned block, float* table) {
  using W = typename Vec<V>::type;
  const FillArgs& f = p.fill;
  const int half = p.rot.num_freqs, head_dim = f.head_dim, tpp = f.tokens_per_page;
  const int heads = p.hq + (p.src_k.data ? f.num_kv_heads : 0);
  const int split = (int)(block % (unsigned)p.head_splits);
  const long long t0 = (long long)(block / (unsigned)p.head_splits) * p.block_tokens;
  const int tokens = (int)min((long long)p.block_tokens, f.num_tokens - t0);
  const int per_split = (heads + p.head_splits - 1) / p.head_splits;
  const int head0 = split * per_split, head1 = min(heads, head0 + per_split);
  if (head0 >= head1) return;
  // thread: unit and token of its pair, and every step-th head from its own
  const int units = (head_dim + 2 * V - 1) / (2 * V), pairs = units * tokens;
  const int step = pairs < kThreads ? kThreads / pairs : 1;
  constexpr int kBatch = 2;  // heads at a time (four: 92 -> 100 us for 16384 tokens, the registers cost resident blocks)
  Elems<T, V> a[kBatch], b[kBatch];
  auto load = [&](const Unit<V, ADJACENT>& u, long long t, int h0) {
    const T* q_row = static_cast<const T*>(p.src_q.data) + t * p.src_q.token_stride;
    const T* k_row = static_cast<const T*>(p.src_k.data) + t * p.src_k.token_stride;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * step;
      if (h >= head1) break;
      const T* src = h < p.hq ? q_row + h * p.src_q.head_stride : k_row + (h - p.hq) * p.src_k.head_stride;
      a[k].v = *reinterpret_cast<const W*>(src + u.first);
      if (u.second >= 0) b[k].v = *reinterpret_cast<const W*>(src + u.second);
    }
  };
  // the first heads travel while the angles are computed
  int i = threadIdx.x;
  if (i < pairs * step) {
    const int j = i / pairs, pair = i - j * pairs, tl = pair / units;
    load(Unit<V, ADJACENT>(pair - tl * units, half, head_dim), t0 + tl, head0 + j);
  }
  for (int e = threadIdx.x; e < tokens * half; e += kThreads) {
    const int t = e / half, k = e - t * half;
    const float2 cs = cos_sin(p.rot, t0 + t, k);
    table[2 * t * half + k] = cs.x;
    table[(2 * t + 1) * half + k] = cs.y;
  }
  __syncthreads();

  for (bool loaded = true; i < pairs * step; i += kThreads) {
    const int j = i / pairs, pair = i - j * pairs;
    const int tl = pair / units, ui = pair - tl * units;
    const long long t = t0 + tl;
    const Unit<V, ADJACENT> u(ui, half, head_dim);
    Angles<V> g;
    if (u.turns) {
      const float *c = table + 2 * tl * half + V * ui, *sn = c + half;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        g.c[e] = c[e];
        g.s[e] = sn[e];
      }
    }
    T* q_out = static_cast<T*>(p.q_out) + t * p.q_out_token_stride;
    // element e of a key lies in chunk e / 8 of its (page, head) block, at [chunk][slot][e % 8]
    long long page = -1;
    int slot = 0;
    if (head1 > p.hq) destination(f, t, page, slot);
    T* pool = static_cast<T*>(f.k_pool) + page * f.num_kv_heads * head_dim * tpp;
    const int o1 = ((u.first >> 3) * tpp + slot) * 8 + (u.first & 7);
    const int o2 = u.second >= 0 ? ((u.second >> 3) * tpp + slot) * 8 + (u.second & 7) : 0;
    for (int h0 = head0 + j; h0 < head1; h0 += kBatch * step) {
      if (!loaded) load(u, t, h0);
      loaded = false;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int h = h0 + k * step;
        if (h >= head1) break;
        if (u.turns) turn<T, V, ADJACENT>(a[k], b[k], g);
        if (h < p.hq) {
          T* o = q_out + h * p.q_out_head_stride;
          *reinterpret_cast<W*>(o + u.first) = a[k].v;
          if (u.second >= 0) *reinterpret_cast<W*>(o + u.second) = b[k].v;
        } else if (page >= 0) {
          T* o = pool + (long long)(h - p.hq) * head_dim * tpp;
          *reinterpret_cast<W*>(o + o1) = a[k].v;
          if (u.second >= 0) *reinterpret_cast<W*>(o + o2) = b[k].v;
        }
      }
    }
  }
}

// One V block: tokens [t0, t0 + 64) of one head.  A staged row is padded to whole groups of eight 16-byte chunks, and chunk c
// of row r sits at c ^ swizzle(r): the eight rows one ldmatrix phase reads are tokens b + 8 t (b < 2, t < 4), which the
// swizzle sends to eight different banks.
__device__ __forceinline__ int row_swizzle(int row) { return (row & 1) | (((row >> 3) & 3) << 1); }

__device__ __forceinline__ void move_values(const RotaryParams& p, unsigned block, unsigned char* smem) {
  const FillArgs& f = p.fill;
  __shared__ long long s_page[kTileTokens + 1];  // entry i: token t0 - 1 + i
  __shared__ int s_slot[kTileTokens + 1];
  __shared__ unsigned char s_cont[kTileTokens + 1];  // token t0 + i continues the octet run of its predecessor
  __shared__ unsigned char s_octet[kTokensPerTile];  // first tokens of the full octets
  __shared__ unsigned char s_single[kTileTokens];    // tokens stored one by one
  __shared__ int s_num_octets, s_num_singles;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = (int)(block % (unsigned)f.num_kv_heads);
  const long long t0 = (long long)(block / (unsigned)f.num_kv_heads) * p.v_tokens;
  const int rows = (int)min((long long)p.v_tokens + 7, f.num_tokens - t0);
  const int owned = min(rows, p.v_tokens);
  const int chunks = f.head_dim >> 3, pitch = (chunks + 7) / 8 * 128;
  const uint16_t* src = static_cast<const uint16_t*>(p.src_v.data) + t0 * p.src_v.token_stride + head * p.src_v.head_stride;
  const uint32_t sbase = smem_u32(smem);

  // the rows do not depend on where they go: their copies travel while the destinations are looked up
  if (p.v_vec) {
    for (int i = tid; i < rows * chunks; i += kThreads) {
      const int r = i / chunks, c = i - r * chunks;
      cp_async_16(smem + r * pitch + ((c ^ row_swizzle(r)) << 4), src + r * p.src_v.token_stride + c * 8);
    }
  } else {
    for (int i = tid; i < rows * f.head_dim; i += kThreads) {
      const int r = i / f.head_dim, d = i - r * f.head_dim;
      *reinterpret_cast<uint16_t*>(smem + r * pitch + (((d >> 3) ^ row_swizzle(r)) << 4) + (d & 7) * 2) = src[r * p.src_v.token_stride + d];
    }
  }
  if (tid <= kTileTokens) {
    const long long t = t0 - 1 + tid;
    long long page = -1;
    int slot = 0;
    if (t >= 0 && tid <= rows) destination(f, t, page, slot);
    s_page[tid] = page;
    s_slot[tid] = slot;
  }
  if (tid == 0) s_num_octets = s_num_singles = 0;
  __syncthreads();
  if (tid < kTileTokens) {
    const int i = tid + 1;
    s_cont[tid] = s_page[i] >= 0 && s_page[i - 1] == s_page[i] && s_slot[i - 1] + 1 == s_slot[i] && (s_slot[i] & 7) != 0;
  }
  __syncthreads();
  if (tid < owned && s_page[tid + 1] >= 0 && !s_cont[tid]) {
    int n = 1;
    while (n < 8 && tid + n < rows && s_cont[tid + n]) ++n;
    // (16-byte stores need the eight slots to start at a multiple of eight and the rows of the pool to be 16-byte aligned)
    if (n == 8 && (s_slot[tid + 1] & 7) == 0 && (f.tokens_per_page & 7) == 0) {
      s_octet[atomicAdd(&s_num_octets, 1)] = (unsigned char)tid;
    } else {
      const int at = atomicAdd(&s_num_singles, n);
      for (int k = 0; k < n; ++k) s_single[at + k] = (unsigned char)(tid + k);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  uint16_t* pool = static_cast<uint16_t*>(f.v_pool) + (long long)head * f.head_dim * f.tokens_per_page;
  const long long page_elems = (long long)f.num_kv_heads * f.head_dim * f.tokens_per_page;
  const int num_octets = s_num_octets, num_singles = s_num_singles;
  const int quads = (num_octets + 3) >> 2;
  for (int w = warp; w < quads * chunks; w += kThreads / 32) {
    const int q4 = w / chunks, c = w - q4 * chunks;
    const int k = lane >> 3, row_t = (lane & 7) >> 1, row_b = lane & 1;
    const int row = s_octet[min(4 * q4 + row_t, num_octets - 1)] + 2 * k + row_b;
    uint32_t v[4];
    ldmatrix_x4_trans(v, sbase + row * pitch + ((c ^ row_swizzle(row)) << 4));
    const int mine = 4 * q4 + (lane & 3), d = 8 * c + (lane >> 2);
    if (mine < num_octets) {
      const int first = s_octet[mine] + 1;
      *reinterpret_cast<uint4*>(pool + s_page[first] * page_elems + (long long)d * f.tokens_per_page + s_slot[first]) =
          make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
  for (int i = tid; i < num_singles * f.head_dim; i += kThreads) {
    const int n = i / f.head_dim, d = i - n * f.head_dim;
    const int row = s_single[n];
    pool[s_page[row + 1] * page_elems + (long long)d * f.tokens_per_page + s_slot[row + 1]] =
        *reinterpret_cast<const uint16_t*>(smem + row * pitch + (((d >> 3) ^ row_swizzle(row)) << 4) + (d & 7) * 2);
  }
}

template <typename T, int V, bool ADJACENT>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ __align__(128) unsigned char rotary_smem[];
  if (blockIdx.x < p.v_blocks)
    move_values(p, blockIdx.x, rotary_smem);
  else
    rotate<T, V, ADJACENT>(p, blockIdx.x - p.v_blocks, reinterpret_cast<float*>(rotary_smem));
}

bool aligned_rows(const void* data, long long token_stride, long long head_stride, int bytes) {
  return reinterpret_cast<uintptr_t>(data) % bytes == 0 && (token_stride * 2) % bytes == 0 && (head_stride * 2) % bytes == 0;
}

template <typename T, int V, bool ADJACENT>
int launch_inst(const RotaryParams& p, unsigned long long rotating, size_t smem, cudaStream_t stream) {
  const unsigned long long blocks = rotating + p.v_blocks;
  if (blocks > 0x7fffffffULL) {
    set_error("rotary: too many tokens for one launch");
    return -2;
  }
  rotary_kernel<T, V, ADJACENT><<<(unsigned)blocks, kThreads, smem, stream>>>(p);
  return (int)cudaGetLastError();
}

template <typename T>
int launch_typed(const RotaryParams& p, int vec, unsigned long long rotating, size_t smem, cudaStream_t stream) {
  const bool adjacent = p.rot.pairing == 1;
  if (vec == 8) return adjacent ? launch_inst<T, 8, true>(p, rotating, smem, stream) : launch_inst<T, 8, false>(p, rotating, smem, stream);
  if (vec == 4) return adjacent ? launch_inst<T, 4, true>(p, rotating, smem, stream) : launch_inst<T, 4, false>(p, rotating, smem, stream);
  return adjacent ? launch_inst<T, 1, true>(p, rotating, smem, stream) : launch_inst<T, 1, false>(p, rotating, smem, stream);
}

}  // namespace

int launch_rotary(const RotaryArgs& a, cudaStream_t stream) {
  RotaryParams p{};
  p.rot = a.rot;
  p.src_q = a.q;
  p.src_k = a.k;
  p.src_v = a.v;
  p.q_out = a.q_out.data;
  p.q_out_token_stride = a.q_out.token_stride;
  p.q_out_head_stride = a.q_out.head_stride;
  p.fill = a.fill;
  p.hq = a.q.data ? a.num_q_heads : 0;
  const int d = a.fill.head_dim, half = a.rot.num_freqs;
  const long long tokens = a.fill.num_tokens;
  // The widest vector that divides the row, the rotated half and every stride: 16 bytes for all common layouts, 8 for
  // rotated halves like 20, single elements for the rest.
  int vec = 1;
  for (int v : {8, 4}) {
    bool ok = d % v == 0 && half % v == 0;
    if (a.q.data) ok = ok && aligned_rows(a.q.data, a.q.token_stride, a.q.head_stride, 2 * v) &&
                       aligned_rows(a.q_out.data, a.q_out.token_stride, a.q_out.head_stride, 2 * v);
    if (a.k.data) ok = ok && aligned_rows(a.k.data, a.k.token_stride, a.k.head_stride, 2 * v);
    if (ok) {
      vec = v;
      break;
    }
  }
  const int heads = p.hq + (a.k.data ? a.fill.num_kv_heads : 0);
  // Sixteen tokens share a block once that gives every SM one; below, a token has blocks of its own, one per as many heads as
  // its threads hold at once while the GPU has room for them.
  const long long sms = cached_sm_count();
  const size_t token_bytes = (size_t)2 * half * sizeof(float);
  p.block_tokens = tokens >= kTokensPerBlock * sms && kTokensPerBlock * token_bytes <= kTableBytes ? kTokensPerBlock : 1;
  const long long groups = (tokens + p.block_tokens - 1) / p.block_tokens;
  const int units = (d + 2 * vec - 1) / (2 * vec);
  const int at_once = kThreads / units > 1 ? kThreads / units : 1;
  const long long splits_wanted = (heads + at_once - 1) / at_once, splits_room = 4 * sms / groups;
  p.head_splits = (int)(splits_room < 1 ? 1 : (splits_room < splits_wanted ? splits_room : splits_wanted));
  size_t smem = p.block_tokens * token_bytes;
  if (a.k.data) {
    p.v_tokens = tokens * a.fill.num_kv_heads >= kTokensPerTile * sms ? kTokensPerTile : 8;
    p.v_blocks = (unsigned)((tokens + p.v_tokens - 1) / p.v_tokens * a.fill.num_kv_heads);
    p.v_vec = aligned_rows(a.v.data, a.v.token_stride, a.v.head_stride, 16) ? 1 : 0;
    const size_t rows = (size_t)(tokens < p.v_tokens + 7 ? tokens : p.v_tokens + 7) * ((d / 8 + 7) / 8 * 128);
    if (rows > smem) smem = rows;
  }
  const unsigned long long rotating = (unsigned long long)groups * p.head_splits;
  return a.dtype == 0 ? launch_typed<__half>(p, vec, rotating, smem, stream) : launch_typed<__nv_bfloat16>(p, vec, rotating, smem, stream);
}

}  // namespace pal
