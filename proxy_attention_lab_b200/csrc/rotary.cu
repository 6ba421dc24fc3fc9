// Rotary position embedding for sm_100a: the rotation of queries / keys by one to four position axes, alone
// (rotary_embedding) or on the way into the page pools (fill_kv_pages_rotary).
//
// Mathematics.  Frequency i (of R / 2) turns one pair of elements (a, b) of every head by the angle
// t = position[axis(i)] * inv_freq[i]:   a' = m (a cos t - b sin t),   b' = m (b cos t + a sin t),
// with (a, b) = elements (i, i + R/2) or (2i, 2i + 1), and m a common magnitude.  Elements past R pass through.
// The angle of a far position is large (position 10^6 times frequency 1), and its fp32 product would be off by up to
// 2^-24 * 10^6 = 0.06 rad, so product and reduction to a fraction of a turn are taken in fp64 (exact product for
// positions below 2^29); the fraction, at most half a turn, is then good to 2^-25 turns in fp32 and sincospif does the rest.
//
// Bound: memory.  A rotated element costs 4 bytes of traffic and ~3 flops; the angle, ~60 instructions, is shared by all
// heads of a token.  So a thread owns one unit - 2 V elements of a head row, V frequencies - of one token, computes its V
// sines and cosines once into registers and walks over heads with 16-byte loads and stores (V = 8).  How many heads a thread
// takes is chosen so that the grid fills the GPU first (a few tokens: one head per thread) and shares angles second.
//
// fill_kv_pages_rotary is one launch of blocks in three roles: rotate the queries into their output, rotate the keys into
// the K pool, move the values into the V pool.
//   K pool [P, Hkv, D/8, TPP, 8]: a unit is whole 16-byte chunks; eight lanes take eight consecutive tokens, so that a warp
//     writes runs of 128 contiguous bytes per chunk while it reads 64 bytes of each token row.
//   V pool [P, Hkv, D, TPP]: eight consecutive slots of a page are 16 contiguous bytes of a head-dim row.  A block stages 64
//     tokens (and the 7 that follow them) of one head in shared memory and finds the octets: runs of eight tokens that fill
//     an aligned group of eight slots.  An octet belongs to the block that holds its first token, hence the halo: prompts
//     start anywhere in a page, and cutting octets at block borders would turn a fifth of the stores into 2-byte ones.
//     ldmatrix.trans does the transposition: its row addresses are free, so row 2 t + b of matrix k is given the address of
//     token 2 k + b of octet t, and each lane receives the eight tokens of one head-dim element of octet t in four
//     registers - one 16-byte store.  The rest (single tokens, ends of runs) leaves in 2-byte stores.
#include "common.cuh"
#include "launch.h"

namespace pal {
namespace {

constexpr int kThreads = 256;
constexpr int kTokensPerTile = 64;               // list tokens a V block owns
constexpr int kTileTokens = kTokensPerTile + 7;  // ... and stages: the octet that starts at its last token ends 7 later
constexpr int kKeyLanes = 8;                     // consecutive tokens on consecutive lanes in the K role

struct RotaryParams {
  RotationArgs rot;
  RowsView src_q, src_k, src_v;
  void* q_out;
  long long q_out_token_stride, q_out_head_stride;
  FillArgs fill;
  int hq;               // query heads to rotate (0 = none)
  int q_step, k_step;   // threads that share a (token, unit): thread j takes heads j, j + step, ...
  unsigned q_blocks, k_blocks, v_blocks;
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

template <int V>
struct Angles {
  float c[V], s[V];
  __device__ __forceinline__ void compute(const RotationArgs& r, long long token, int i0) {
    int axis = -1;
    double pos = 0.0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int a = axis_of(r, i0 + e);
      if (a != axis) {
        axis = a;
        const long long at = a * r.positions_axis_stride + token;
        pos = r.positions_64bit ? (double)static_cast<const long long*>(r.positions)[at] : (double)static_cast<const int*>(r.positions)[at];
      }
      double turns = pos * (double)r.inv_freq[i0 + e] * 0.15915494309189533577;  // 1 / (2 pi)
      turns -= rint(turns);
      float sn, cs;
      sincospif(2.0f * (float)turns, &sn, &cs);
      c[e] = cs * r.magnitude;
      s[e] = sn * r.magnitude;
    }
  }
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

// (page, slot) of token t, or page = -1 when the token is skipped: the rules of fill_kv_pages
__device__ __forceinline__ void destination(const FillArgs& f, long long t, long long& page, int& slot) {
  page = -1;
  slot = 0;
  if (f.slot_mapping) {
    const long long s = f.slot_mapping[t];
    if (s < 0 || s >= f.num_pages * f.tokens_per_page) return;
    page = s / f.tokens_per_page;
    slot = (int)(s - page * f.tokens_per_page);
  } else {
    const uint32_t seq = static_cast<const uint32_t*>(f.query_to_seq_map)[t];
    const int pos = f.write_positions[t];
    if (pos < 0 || seq >= (uint32_t)f.num_seqs) return;
    const int block = pos / f.tokens_per_page;
    if (block >= f.max_pages_per_seq) return;
    const long long pg = static_cast<const uint32_t*>(f.page_table)[(long long)seq * f.max_pages_per_seq + block];
    if (pg >= f.num_pages) return;
    page = pg;
    slot = pos - block * f.tokens_per_page;
  }
}

// Heads j, j + step, ... of one (token, unit), four at a time so that eight loads are in flight before the first use.
template <typename T, int V, bool ADJACENT, typename Store>
__device__ __forceinline__ void walk_heads(const T* row, long long head_stride, int heads, int j, int step, const Unit<V, ADJACENT>& u,
                                           const Angles<V>& g, Store&& store) {
  using W = typename Vec<V>::type;
  constexpr int kBatch = 4;
  for (int h0 = j; h0 < heads; h0 += kBatch * step) {
    Elems<T, V> a[kBatch], b[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * step;
      if (h >= heads) break;
      const T* p = row + h * head_stride;
      a[k].v = *reinterpret_cast<const W*>(p + u.first);
      if (u.second >= 0) b[k].v = *reinterpret_cast<const W*>(p + u.second);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * step;
      if (h >= heads) break;
      if (u.turns) turn<T, V, ADJACENT>(a[k], b[k], g);
      store(h, a[k], b[k]);
    }
  }
}

template <typename T, int V, bool ADJACENT>
__device__ __forceinline__ void rotate_queries(const RotaryParams& p, long long tid, int units) {
  const int head_dim = p.fill.head_dim, half = p.rot.num_freqs;
  const int ui = (int)(tid % units);
  const long long r = tid / units;
  const int j = (int)(r % p.q_step);
  const long long t = r / p.q_step;
  if (t >= p.fill.num_tokens) return;
  const Unit<V, ADJACENT> u(ui, half, head_dim);
  Angles<V> g;
  if (u.turns) g.compute(p.rot, t, V * ui);
  using W = typename Vec<V>::type;
  T* out = static_cast<T*>(p.q_out) + t * p.q_out_token_stride;
  walk_heads<T, V, ADJACENT>(static_cast<const T*>(p.src_q.data) + t * p.src_q.token_stride, p.src_q.head_stride, p.hq, j, p.q_step, u, g,
                             [&](int h, const Elems<T, V>& a, const Elems<T, V>& b) {
                               T* o = out + h * p.q_out_head_stride;
                               *reinterpret_cast<W*>(o + u.first) = a.v;
                               if (u.second >= 0) *reinterpret_cast<W*>(o + u.second) = b.v;
                             });
}

template <typename T, int V, bool ADJACENT>
__device__ __forceinline__ void rotate_keys(const RotaryParams& p, long long tid, int units) {
  const FillArgs& f = p.fill;
  const int half = p.rot.num_freqs;
  const int tl = (int)(tid % kKeyLanes);
  long long r = tid / kKeyLanes;
  const int ui = (int)(r % units);
  r /= units;
  const int j = (int)(r % p.k_step);
  const long long t = r / p.k_step * kKeyLanes + tl;
  if (t >= f.num_tokens) return;
  long long page;
  int slot;
  destination(f, t, page, slot);
  if (page < 0) return;
  const Unit<V, ADJACENT> u(ui, half, f.head_dim);
  Angles<V> g;
  if (u.turns) g.compute(p.rot, t, V * ui);
  using W = typename Vec<V>::type;
  const int tpp = f.tokens_per_page;
  // element e of a head lies in chunk e / 8 at [chunk][slot][e % 8]
  const long long o1 = ((long long)(u.first >> 3) * tpp + slot) * 8 + (u.first & 7);
  const long long o2 = u.second >= 0 ? ((long long)(u.second >> 3) * tpp + slot) * 8 + (u.second & 7) : 0;
  T* pool = static_cast<T*>(f.k_pool) + page * f.num_kv_heads * f.head_dim * tpp;
  walk_heads<T, V, ADJACENT>(static_cast<const T*>(p.src_k.data) + t * p.src_k.token_stride, p.src_k.head_stride, f.num_kv_heads, j, p.k_step,
                             u, g, [&](int h, const Elems<T, V>& a, const Elems<T, V>& b) {
                               T* o = pool + (long long)h * f.head_dim * tpp;
                               *reinterpret_cast<W*>(o + o1) = a.v;
                               if (u.second >= 0) *reinterpret_cast<W*>(o + o2) = b.v;
                             });
}

__device__ __forceinline__ void copy_async_16(uint32_t smem_dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_transposed(uint32_t (&r)[4], uint32_t saddr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(saddr)
               : "memory");
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
  const long long t0 = (long long)(block / (unsigned)f.num_kv_heads) * kTokensPerTile;
  const int rows = (int)min((long long)kTileTokens, f.num_tokens - t0);
  const int owned = min(rows, kTokensPerTile);
  const int chunks = f.head_dim >> 3, pitch = (chunks + 7) / 8 * 128;
  const uint16_t* src = static_cast<const uint16_t*>(p.src_v.data) + t0 * p.src_v.token_stride + head * p.src_v.head_stride;
  const uint32_t sbase = smem_u32(smem);

  // the rows do not depend on where they go: their copies travel while the destinations are looked up
  if (p.v_vec) {
    for (int i = tid; i < rows * chunks; i += kThreads) {
      const int r = i / chunks, c = i - r * chunks;
      copy_async_16(sbase + r * pitch + ((c ^ row_swizzle(r)) << 4), src + r * p.src_v.token_stride + c * 8);
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
    ldmatrix_x4_transposed(v, sbase + row * pitch + ((c ^ row_swizzle(row)) << 4));
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
  const int units = (p.fill.head_dim + 2 * V - 1) / (2 * V);
  unsigned b = blockIdx.x;
  if (b < p.v_blocks) {
    move_values(p, b, rotary_smem);
    return;
  }
  b -= p.v_blocks;
  if (b < p.k_blocks) {
    rotate_keys<T, V, ADJACENT>(p, (long long)b * kThreads + threadIdx.x, units);
    return;
  }
  b -= p.k_blocks;
  rotate_queries<T, V, ADJACENT>(p, (long long)b * kThreads + threadIdx.x, units);
}

bool aligned_rows(const void* data, long long token_stride, long long head_stride, int bytes) {
  return reinterpret_cast<uintptr_t>(data) % bytes == 0 && (token_stride * 2) % bytes == 0 && (head_stride * 2) % bytes == 0;
}

// Threads that share a (token, unit): as many as it takes for every SM to hold 1024 threads, at most one per head.  With
// more tokens than that a thread takes several heads and the angles are computed once for them.
int head_step(long long token_units, int heads) {
  const long long want = 148LL * 1024;
  long long step = (want + token_units - 1) / token_units;
  return (int)(step < 1 ? 1 : (step > heads ? heads : step));
}

template <typename T, int V, bool ADJACENT>
int launch_inst(const RotaryParams& p, size_t smem, cudaStream_t stream) {
  const unsigned long long blocks = (unsigned long long)p.q_blocks + p.k_blocks + p.v_blocks;
  if (blocks > 0x7fffffffULL) {
    set_error("rotary: too many tokens for one launch");
    return -2;
  }
  rotary_kernel<T, V, ADJACENT><<<(unsigned)blocks, kThreads, smem, stream>>>(p);
  return (int)cudaGetLastError();
}

template <typename T>
int launch_typed(const RotaryParams& p, int vec, size_t smem, cudaStream_t stream) {
  const bool adjacent = p.rot.pairing == 1;
  if (vec == 8) return adjacent ? launch_inst<T, 8, true>(p, smem, stream) : launch_inst<T, 8, false>(p, smem, stream);
  if (vec == 4) return adjacent ? launch_inst<T, 4, true>(p, smem, stream) : launch_inst<T, 4, false>(p, smem, stream);
  return adjacent ? launch_inst<T, 1, true>(p, smem, stream) : launch_inst<T, 1, false>(p, smem, stream);
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
  const long long units = (d + 2 * vec - 1) / (2 * vec);
  size_t smem = 0;
  auto blocks_for = [](long long threads) { return (unsigned)((threads + kThreads - 1) / kThreads); };
  if (p.hq > 0) {
    p.q_step = head_step(tokens * units, p.hq);
    p.q_blocks = blocks_for(tokens * units * p.q_step);
  }
  if (a.k.data) {
    const long long groups = (tokens + kKeyLanes - 1) / kKeyLanes;
    p.k_step = head_step(groups * kKeyLanes * units, a.fill.num_kv_heads);
    p.k_blocks = blocks_for(groups * kKeyLanes * units * p.k_step);
    p.v_blocks = (unsigned)((tokens + kTokensPerTile - 1) / kTokensPerTile * a.fill.num_kv_heads);
    p.v_vec = aligned_rows(a.v.data, a.v.token_stride, a.v.head_stride, 16) ? 1 : 0;
    const int rows = (int)(tokens < kTileTokens ? tokens : kTileTokens);
    smem = (size_t)rows * ((d / 8 + 7) / 8 * 128);
  }
  return a.dtype == 0 ? launch_typed<__half>(p, vec, smem, stream) : launch_typed<__nv_bfloat16>(p, vec, smem, stream);
}

}  // namespace pal
