// Sequences that share a history: new tokens into a paged cache (skv_append_pages) and attention of
// a batch whose sequences all see one prefix and then pages of their own (skv_attend_shared).
//
// A page is a frame slot with a batch of one: K [pages][H][Tp][128], V [pages][H][128][Tp], T
// tokens of a page in use (Tp = T rounded up to 64).  A sequence's token i lies at offset i % T of
// page tables[b][i / T]; page numbers outside the pool are pages that are not there: nothing is
// written to them and their keys are not seen.
#include <utility>

#include "skv_rowops.h"

namespace skv {

namespace {

// ---------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------
struct Pages {
  const int32_t* tables;
  int64_t table_st;
  int64_t capacity;  // tokens of a table: width * T, below 2^31
  int n_pages, T, Tp, heads;
  const int32_t* lengths;
  const int32_t* new_lens;

  // tokens of sequence b with the new ones, and the new ones among its `rows` rows
  __device__ int fresh(int b, int rows) const {
    if (new_lens == nullptr) return rows;
    const int n = new_lens[b];
    return n < 0 ? 0 : n > rows ? rows : n;
  }
  __device__ int64_t first(int b, int n) const { return (int64_t)lengths[b] - n; }
};

struct AppendPagesArgs {
  Pages pg;
  const void *q, *k, *v;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  void* q_out;
  int64_t o_sb, o_st, o_sh;
  void *k_pool, *v_pool;
  const void *wq, *wk;
  int wq_dtype, wk_dtype, norm_q, norm_k, q_heads, q_blocks, k_blocks;
  float eps_q, eps_k;
  const float *cos, *sin;
  int64_t tab_st, tab_rows;
  const void* pos;
  int64_t pos_sb, pos_st, pos0;
  int pos64, half, batch, rows;
  int n_units_q, n_units, n_unit_groups;  // (token, head block) units of q and of q and k
  int v_tiles;                            // tiles of pages that a sequence's tokens may reach
};

// Where a sequence's token `own` lies: its page (-1 where there is none) and its place in it.
struct Place {
  int64_t page;
  int off;
};
__device__ inline Place place_of(const Pages& pg, int b, int64_t own) {
  if (own < 0 || own >= pg.capacity) return Place{-1, 0};
  const int p = (int)own / pg.T, id = pg.tables[b * pg.table_st + p];
  return Place{id < 0 || id >= pg.n_pages ? -1 : id, (int)own - p * pg.T};
}

// V of the tokens that one 64-token tile of a page takes: rows in through LDS, out as pieces of 8
// tokens of a channel (16 B) where all 8 are new, token by token at the ends, past the caches (as the rows of K
// and q: together 77 -> 65 us for the eight sequences below).  A call of one token a
// sequence goes the same way: a wave per token that stores its channels straight away takes as long
// (128 sequences of 8 heads 6.6 us either way; 64 sequences of 8 tokens 9.9 us, by tiles 9.2).
template <typename T>
__device__ inline void v_tile(const AppendPagesArgs& a, int unit, uint32_t (&buf)[kTile][65]) {
  const int j = unit % a.v_tiles, bh = unit / a.v_tiles;
  const int h = bh % a.pg.heads, b = bh / a.pg.heads;
  const int n = a.pg.fresh(b, a.rows);
  const int64_t first = a.pg.first(b, n), end = first + n < a.pg.capacity ? first + n : a.pg.capacity;
  if (end <= (first > 0 ? first : 0)) return;
  const int from = first > 0 ? (int)first : 0, to = (int)end;
  const int per_page = (a.pg.T + kTile - 1) / kTile;
  const int p0 = from / a.pg.T, tile = p0 * per_page + (from - p0 * a.pg.T) / kTile + j;
  const int p = tile / per_page, t0 = (tile - p * per_page) * kTile;  // its page, its first token there
  const int64_t base = (int64_t)p * a.pg.T + t0;                      // and that token's own index
  if (base >= to) return;
  const int cap = a.pg.T - t0 < kTile ? a.pg.T - t0 : kTile;
  const int lo = from > base ? from - (int)base : 0, hi = to - (int)base < cap ? to - (int)base : cap;
  if (lo >= hi) return;
  const int id = a.pg.tables[b * a.pg.table_st + p];
  if (id < 0 || id >= a.pg.n_pages) return;
  const int64_t row0 = base - first;  // the call's row of the tile's first token
  const int tid = threadIdx.x, c = tid & 15;
  const T* v = static_cast<const T*>(a.v) + b * a.v_sb + h * a.v_sh + 8 * c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (tid >> 4) + 16 * i;
    if (r >= lo && r < hi) {
      const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(v + (row0 + r) * a.v_st));
#pragma unroll
      for (int e = 0; e < 4; ++e) buf[r][4 * c + e] = w[e];
    }
  }
  __syncthreads();
  uint16_t* o = static_cast<uint16_t*>(a.v_pool) +
                ((int64_t)id * a.pg.heads + h) * kHeadDim * (int64_t)a.pg.Tp + t0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int piece = tid & 7, pair = (tid >> 3) + 32 * i;  // 8 tokens of channels 2 pair, 2 pair + 1
    const int r0 = 8 * piece;
    if (r0 >= hi || r0 + 8 <= lo) continue;
    u32x4 even, odd;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = buf[r0 + 2 * e][pair], y = buf[r0 + 2 * e + 1][pair];
      even[e] = (x & 0xffffu) | (y << 16);
      odd[e] = (x >> 16) | (y & 0xffff0000u);
    }
    uint16_t* p0w = o + (int64_t)(2 * pair) * a.pg.Tp + r0;
    uint16_t* p1w = p0w + a.pg.Tp;
    if (r0 >= lo && r0 + 8 <= hi) {
      __builtin_nontemporal_store(even, reinterpret_cast<u32x4*>(p0w));
      __builtin_nontemporal_store(odd, reinterpret_cast<u32x4*>(p1w));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (r0 + e >= lo && r0 + e < hi) {
          p0w[e] = (uint16_t)(even[e / 2] >> (16 * (e & 1)));
          p1w[e] = (uint16_t)(odd[e / 2] >> (16 * (e & 1)));
        }
    }
  }
}

// Workgroups [0, n_unit_groups): 16 (token, head block) units each of q and then of k; the rest:
// V, a tile of a page each.  One launch does all of it: it is bound by bytes where there are many tokens
// (eight padded sequences of up to 1560 tokens, 24 heads, zero rows of the padding included: 151 MB read and
// 186 written in 58 us, 5.8 TB/s with part of the input in the last cache) and by its launch where there are few (3.9 us for one token of 12 heads, 5.6 for 64 of 32 + 8).
template <typename T, bool INTER>
__global__ __launch_bounds__(256) void append_pages_kernel(AppendPagesArgs a) {
  __shared__ uint32_t buf[kTile][65];
  if ((int)blockIdx.x >= a.n_unit_groups) {
    v_tile<T>(a, (int)blockIdx.x - a.n_unit_groups, buf);
    return;
  }
  const int lane64 = threadIdx.x & 63, c = 8 * (lane64 & 15);
  int unit = (int)blockIdx.x * 16 + (threadIdx.x >> 4);
  const TurnLane<INTER> lane(a.half, lane64);
  const bool live = unit < a.n_units;
  const bool is_q = live && unit < a.n_units_q;
  unit = !live ? 0 : is_q ? unit : unit - a.n_units_q;
  const int blocks = is_q ? a.q_blocks : a.k_blocks, heads = is_q ? a.q_heads : a.pg.heads;
  const int h0 = unit % blocks * kHeadBlock, bl = unit / blocks;
  const int row = bl % a.rows, b = bl / a.rows;
  const int64_t st = is_q ? a.q_sh : a.k_sh;
  const T* x = is_q ? static_cast<const T*>(a.q) + b * a.q_sb + row * a.q_st
                    : static_cast<const T*>(a.k) + b * a.k_sb + row * a.k_st;
  const int n = a.pg.fresh(b, a.rows);
  const bool token = live && row < n;
  Raw8<T> raw[kHeadBlock];
#pragma unroll
  for (int i = 0; i < kHeadBlock; ++i)
    raw[i] = token && h0 + i < heads ? Raw8<T>::load(x + (h0 + i) * st + c) : Raw8<T>::zero();
  const int64_t own = a.pg.first(b, n) + row;
  int64_t pos = a.pos0 + own;
  if (a.pos != nullptr) {
    const int64_t i = b * a.pos_sb + row * a.pos_st;
    pos = a.pos0 + (a.pos64 ? static_cast<const int64_t*>(a.pos)[i]
                            : (int64_t)static_cast<const int32_t*>(a.pos)[i]);
  }
  Turn<INTER> turn;
  turn.load(a.cos, a.sin, a.tab_st, a.tab_rows, pos, lane);
  const void* wt = is_q ? a.wq : a.wk;
  const int wd = is_q ? a.wq_dtype : a.wk_dtype;
  float w[8], wp[8];
  load_weight8(wt, wd, c, w);
  if constexpr (!INTER) load_weight8(wt, wd, 8 * (lane.partner & 15), wp);
  T* o = nullptr;
  int64_t oh = 0;
  if (is_q) {
    o = static_cast<T*>(a.q_out) + b * a.o_sb + row * a.o_st;
    oh = a.o_sh;
  } else if (token) {
    const Place at = place_of(a.pg, b, own);
    if (at.page >= 0) o = static_cast<T*>(a.k_pool) + (at.page * a.pg.heads * a.pg.Tp + at.off) * kHeadDim;
    oh = (int64_t)a.pg.Tp * kHeadDim;
  }
  const bool norm = is_q ? a.norm_q : a.norm_k;
  const float eps = is_q ? a.eps_q : a.eps_k;
#pragma unroll
  for (int i = 0; i < kHeadBlock; ++i) {
    Raw8<T> z = norm_turn<T, INTER>(raw[i], norm, eps, w, wp, turn, lane);
    if (!token) z = Raw8<T>::zero();  // rows behind a sequence's new tokens
    if (o != nullptr && live && h0 + i < heads) z.store(o + (h0 + i) * oh + c);
  }
}

// ---------------------------------------------------------------------------------------------
// attention
//
// With G = query heads per key head, row m = (b * L + l) * G + g of key head h is query (b, l, h G
// + g).  The prefix's scores are products of its keys with ALL rows of a key head, so its K and V
// are read once for the batch (once per row block); a sequence's own pages meet its own L * G rows.
// Both are split along the keys; every part leaves per row its maximum m, its sum l of exp2(s - m)
// and its unnormalised fp32 output, which merge_kernel joins:
//   out = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p,  m = max m_p.
//
// S^T = K Q^T and O^T = V^T P^T, so a lane holds one row's scores.  The rows of S^T are keys in an
// order that makes the probabilities a lane holds those of neighbouring keys: they are the second
// product's B operand as they stand, and its A operand is 16 B pieces of V rows.
//
// A workgroup of 8 waves has a CU to itself (the tiles take 128 KB of its LDS, a wave up to 256 registers)
// and works on one item: some rows of a key head against a share of the keys.  By the number of rows:
//  * up to 16 stream: every wave takes its own share of the keys, K and V straight from memory to
//    registers.  Bound by bytes: 21 sequences, 12 heads, 7808 keys each, 1 GB in 197 us, 5.1 TB/s.
//  * up to 128: two tiles of 64 keys a round in LDS, four waves of 32 rows on each.  Bound by
//    bytes up to some 64 rows (the same keys 176 us, 5.7 TB/s with some of it in the last cache); 213 us at
//    128 rows.
//  * more: 256 rows, one tile a round, software-pipelined.  Bound by the matrix cores and the power they
//    draw: 1024 rows of 8 heads against 131072 keys 521 us, 1.05 PFLOP/s, where a large library product
//    reaches 1.35; a tile takes 1.45 us with half of the CUs at work and 2.0 with all.  Each 32 x 16 operand
//    is read from LDS by the wave that multiplies it, 256 KB a tile, which takes LDS as long as the products
//    take the matrix cores.
// The limits, both sides measured (us): 4 sequences of 16 rows, 12 heads, 7808 keys 41.6 streaming, 43.0 by
// tiles, and 20 rows of 8 heads against 32760 keys 46.6 and 39.2; 128 rows of those sequences 48.5 by two
// tiles a round, 54.9 by one, and 160 rows 79.6 and 71.6.
// ---------------------------------------------------------------------------------------------
constexpr int kWaves = 8;    // of a workgroup: one workgroup a CU, two waves a SIMD
// rows of a work item that streams (0) or goes by 1 or 2 tiles a round, and how many rows go
constexpr int kind_rows(int kind) { return kind == 0 ? 16 : 32 * kWaves / kind; }
constexpr int kind_of(int64_t rows) { return rows <= 16 ? 0 : rows <= 128 ? 2 : 1; }
constexpr int kStep = 32;    // keys of a streaming step
// Sequences whose padding rows a prefix by tiles leaves out (a search in LDS a lane): 32 sequences of up to
// 16 tokens, half of them padding, 32 + 8 heads, against 32760 keys 342 -> 200 us.
constexpr int kCompact = 1024;
constexpr float kSlack = 8;  // the running maximum may lag the true one by 2^8 (see below)

struct Source {
  const void *k_pool, *v_pool;
  int n_pages, T, Tp;
};

struct SharedArgs {
  const void* q;
  int64_t q_sb, q_st, q_sh;
  void* out;
  int64_t o_sb, o_st, o_sh;
  Source pre, own;
  const int32_t* pre_pages;
  int64_t pre_tokens;
  const int32_t* tables;
  int64_t table_st;
  int width;
  const int32_t* lengths;
  const int32_t* new_lens;
  int batch, rows, heads, group, causal;
  float c;       // softmax_scale * log2(e)
  int M;         // batch * rows * group
  int pre_splits, pre_grid;  // key splits and workgroups of the prefix
  int own_rb, own_splits, own_items, own_waves;  // row blocks of a sequence, key splits; waves of an item
  int direct;    // one part only: workgroups write out themselves
  int both;      // (direct) one sequence, few rows: prefix and own keys in one work item
  float* part_o;   // [part][heads][M][128]
  float2* part_ml; // [part][heads][M]
};

// One work item: rows [m0, m1) of key head h against share `split` of `n_split` of a source's keys.
struct Item {
  const int32_t* list;  // page numbers
  int n_list, h, m0, m1, n_split, split, part;
  const int* tokens;  // rows count new tokens only: exclusive sums of new_lens in LDS (NULL: all rows)
  int n_keys;         // keys that some row sees (below 2^31)
  int open;           // keys that every row sees
  int64_t first_lim;  // keys that row 0 of the sequence sees (causal; each next row one more)
  bool causal;
};

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
  typedef bf16x8 v8;
  __device__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static f32x16 mul(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static constexpr uint32_t kInf = 0x7f80u;
};
template <>
struct Mma<f16> {
  typedef f16x8 v8;
  __device__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ static f32x16 mul(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static constexpr uint32_t kInf = 0x7c00u;
};

__device__ inline float over_groups_max(float x, int first) {  // over the lanes of a row
  for (int s = first; s < 64; s <<= 1) x = fmaxf(x, __shfl_xor(x, s, 64));
  return x;
}
__device__ inline float over_groups_sum(float x, int first) {
  for (int s = first; s < 64; s <<= 1) x += __shfl_xor(x, s, 64);
  return x;
}

// 8 neighbouring values of a V row starting at key `k0`: those at or behind `valid` become zero, so
// that what a page holds there is not multiplied.
template <typename V8>
__device__ inline V8 drop_behind(V8 v, int k0, int valid) {
  u32x4 x = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    x[e] = k0 + 2 * e + 1 < valid ? x[e] : k0 + 2 * e < valid ? x[e] & 0xffffu : 0u;
  return __builtin_bit_cast(V8, x);
}

// Infinities and NaN of a V piece become zero; returns whether there were any.
template <typename T>
__device__ inline bool drop_odd(typename Mma<T>::v8& v) {
  u32x4 x = __builtin_bit_cast(u32x4, v);
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = Mma<T>::kInf, hi = lo << 16;
    if ((x[e] & lo) == lo) x[e] &= 0xffff0000u, odd = true;
    if ((x[e] & hi) == hi) x[e] &= 0xffffu, odd = true;
  }
  v = __builtin_bit_cast(typename Mma<T>::v8, x);
  return odd;
}

// Ones where a piece holds +infinity (kind 0), -infinity (1) or NaN (2), zeros elsewhere.
template <typename T>
__device__ inline typename Mma<T>::v8 marks(typename Mma<T>::v8 v, int kind) {
  u32x4 x = __builtin_bit_cast(u32x4, v);
  const uint32_t one = __builtin_bit_cast(uint16_t, (T)1.0f), want = Mma<T>::kInf | (kind == 1 ? 0x8000u : 0u);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = x[e] & 0xffffu, hi = x[e] >> 16;
    const bool l = kind == 2 ? (lo & 0x7fffu) > Mma<T>::kInf : lo == want;
    const bool h = kind == 2 ? (hi & 0x7fffu) > Mma<T>::kInf : hi == want;
    x[e] = (l ? one : 0u) | (h ? one << 16 : 0u);
  }
  return __builtin_bit_cast(typename Mma<T>::v8, x);
}
__device__ inline float marked(int kind) { return kind == 2 ? __builtin_nanf("") : kind == 1 ? -INFINITY : INFINITY; }

// A work item's page list, 64 entries in a vector register at a time.
struct PageWalk {
  const int32_t* list;
  int n, base, ids;
  __device__ void start(const int32_t* l, int count, int page) {  // then landed(), before the first get()
    list = l;
    n = count;
    load(page);
  }
  __device__ void load(int page) {
    base = page;
    const int i = page + (int)(threadIdx.x & 63);
    ids = i < n ? list[i] : -1;
  }
  // The load's wait stands here, not wherever the paths meet again: there it would drain the tiles under way.
  __device__ void landed() { asm volatile("" : "+v"(ids)); }
  __device__ int get(int page) {
    if (page - base >= 64) {
      load(page);
      landed();
    }
    return __builtin_amdgcn_readlane(ids, page - base);
  }
};

// The steps of `step` keys that n_keys take: whole pages, then what the last page holds.
__device__ inline int steps_of(const Source& src, int n_keys, int step, int per_page) {
  const int full = n_keys / src.T;
  return full * per_page + (n_keys - full * src.T + step - 1) / step;
}

// Where share `i` of `n` begins in `all` steps: shares differ by one step at most.
__device__ inline int share_of(int all, int i, int n) {
  const int each = all / n, more = all - each * n;
  return i * each + (i < more ? i : more);
}

__device__ inline void row_of(const SharedArgs& a, int m, int& b, int& l, int& gh) {
  gh = m % a.group;
  const int bl = m / a.group;
  l = bl % a.rows;
  b = bl / a.rows;
}

// Row m of a work item that counts new tokens only, among all rows.
__device__ inline int all_rows(const SharedArgs& a, const Item& it, int m) {
  if (it.tokens == nullptr) return m;
  const int tk = m / a.group;
  int lo = 0, hi = a.batch;  // the last sequence that begins at or before token tk
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (it.tokens[mid] <= tk ? lo : hi) = mid;
  }
  return (lo * a.rows + tk - it.tokens[lo]) * a.group + m % a.group;
}

__device__ inline int fresh_rows(const SharedArgs& a, int b) {
  if (a.new_lens == nullptr) return a.rows;
  const int n = a.new_lens[b];
  return n < 0 ? 0 : n > a.rows ? a.rows : n;
}

// Four neighbouring output channels d0 .. d0 + 3 of row m, or of its part.
template <typename T>
__device__ inline void put4(const SharedArgs& a, const Item& it, int m, int d0, f32x4 o, float inv, T* dst) {
  if (a.direct) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = inv != 0.0f ? (T)(o[i] * inv) : (T)0.0f;
    *reinterpret_cast<t4*>(dst + d0) = x;
  } else {
    const int64_t at = ((int64_t)it.part * a.heads + it.h) * a.M + m;
    *reinterpret_cast<f32x4*>(a.part_o + at * kHeadDim + d0) = o;
  }
}

// 1 / l of a row that is a new token and sees a key, else 0; and where its output goes.
template <typename T>
__device__ inline float row_out(const SharedArgs& a, const Item& it, int m, float mx, float l, bool first, T** dst) {
  if (!a.direct) {
    if (first) a.part_ml[((int64_t)it.part * a.heads + it.h) * a.M + m] = float2{mx, l};
    return 0.0f;
  }
  int b, row, gh;
  row_of(a, m, b, row, gh);
  *dst = static_cast<T*>(a.out) + b * a.o_sb + row * a.o_st + (int64_t)(it.h * a.group + gh) * a.o_sh;
  return row < fresh_rows(a, b) && l != 0.0f ? 1.0f / l : 0.0f;
}

// Of an item's n_keys, those that the sequence's row l sees.
__device__ inline int keys_seen(const Item& it, int l) {
  if (!it.causal || it.first_lim + l >= it.n_keys) return it.n_keys;
  return it.first_lim + l > 0 ? (int)(it.first_lim + l) : 0;
}

// OWN: a sequence's own keys, which some rows may not see yet (the prefix is seen by all).

// ---- at most 16 rows: a wave streams its own keys, 32 a step, on 16x16x32 MFMAs ----------------
// Row i of S tile t is key (i / 4) * 8 + 4 t + i % 4 of the step; lane (n, g) holds row n's keys
// 8 g .. 8 g + 7.
template <typename T>
struct StreamState {
  typename Mma<T>::v8 q[4];
  f32x4 o[8];
  float mx, sum;
  int m, lim;  // the lane's row (m1 and beyond: none), and how many own keys it sees
};

template <typename T>
__device__ inline void stream_begin(StreamState<T>& w, const SharedArgs& a, const Item& it) {
  const int lane = threadIdx.x & 63;
  w.m = it.m0 + (lane & 15);
  int b, l, gh;
  row_of(a, w.m < it.m1 ? w.m : it.m0, b, l, gh);
  w.lim = keys_seen(it, l);
  const T* p = static_cast<const T*>(a.q) + b * a.q_sb + l * a.q_st +
               (int64_t)(it.h * a.group + gh) * a.q_sh + (lane >> 4) * 8;
#pragma unroll
  for (int st = 0; st < 4; ++st) w.q[st] = *reinterpret_cast<const typename Mma<T>::v8*>(p + st * 32);
#pragma unroll
  for (int d = 0; d < 8; ++d) w.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  w.mx = -INFINITY;
  w.sum = 0.0f;
}

// Steps [s0, s1) of an item's keys.
template <typename T, bool OWN>
__device__ inline void stream_steps(StreamState<T>& w, const SharedArgs& a, const Source& src, const Item& it,
                                    int per_page, int s0, int s1) {
  typedef typename Mma<T>::v8 v8;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  v8 (&q)[4] = w.q;
  f32x4 (&o)[8] = w.o;
  float mx = w.mx, sum = w.sum;
  const int lim = OWN ? w.lim : it.n_keys;
  if (s0 < s1) {
    PageWalk pages;
    int page = s0 / per_page, in_page = s0 - page * per_page;
    pages.start(it.list, it.n_list, page);
    const int k_off = ((n >> 2) * 8 + (n & 3)) * kHeadDim + g * 8, v_off = n * src.Tp + g * 8;
    const T* kp = static_cast<const T*>(src.k_pool);
    const T* vp = static_cast<const T*>(src.v_pool);
    pages.landed();
    int id = pages.get(page);
    v8 kf[2][4];
    auto load_k = [&](int id, int at) {
      // a page that is not there is read as page 0 and masked
      const int64_t pid = id < 0 || id >= src.n_pages ? 0 : id;
      const T* p = kp + ((pid * a.heads + it.h) * src.Tp + at * kStep) * (int64_t)kHeadDim + k_off;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int st = 0; st < 4; ++st)
          kf[t][st] = *reinterpret_cast<const v8*>(p + t * 4 * kHeadDim + st * 32);
    };
    load_k(id, in_page);
    for (int s = s0; s < s1; ++s) {
      const bool there = id >= 0 && id < src.n_pages;
      const int64_t pid = there ? id : 0;
      const T* vb = vp + (pid * a.heads + it.h) * kHeadDim * (int64_t)src.Tp + in_page * kStep;
      v8 vf[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) vf[d] = *reinterpret_cast<const v8*>(vb + d * 16 * (int64_t)src.Tp + v_off);
      const int key0 = page * src.T + in_page * kStep;
      // keys of this step that exist: inside the page, inside the sequence
      int left = it.n_keys - key0;
      const int in_tile = src.T - in_page * kStep;
      if (left > in_tile) left = in_tile;
      const int valid = there ? (left > kStep ? kStep : left) : 0;
      f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int t = 0; t < 2; ++t) sc[t] = Mma<T>::mul(kf[t][st], q[st], sc[t]);
      // the next step's keys load under this step's softmax and second product
      if (s + 1 < s1) {
        if (++in_page == per_page) {
          in_page = 0;
          id = pages.get(++page);
        }
        load_k(id, in_page);
      }
      const bool partial = OWN && key0 + valid > it.open;  // some row may not see all of them
      if (valid < kStep || partial) {
        const int seen = lim - key0, most = seen < valid ? seen : valid;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (8 * g + i >= most) sc[i >> 2][i & 3] = -INFINITY;
#pragma unroll
        for (int d = 0; d < 8; ++d) vf[d] = drop_behind(vf[d], 8 * g, valid);
      }
      float top = sc[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[i >> 2][i & 3]);
      top *= a.c;
      // The maximum only has to keep exp2 in range, so it follows when some row of the wave is 2^8
      // above it: most steps skip the reductions and the rescaling.
      if (__any(top > mx + kSlack)) {
        const float m2 = fmaxf(mx, over_groups_max(top, 16));
        const float f = m2 == mx ? 1.0f : __builtin_amdgcn_exp2f(mx - m2);
        mx = m2;
        sum *= f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] *= f;
      }
      const float ms = mx == -INFINITY ? 0.0f : mx;
      v8 p;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = __builtin_amdgcn_exp2f(sc[i >> 2][i & 3] * a.c - ms);
        sum += e;
        p[i] = (T)e;  // rounded to the pool's type for the matrix product; the sum is of fp32 values
      }
      if (partial) {
        // A key that some rows may not see yet can hold an infinity or a NaN, which 0 * v would spread
        // to them: such values leave the product, and the rows that see one (their probability times a
        // mark is not zero) get it.
        v8 clean[8];
        bool odd = false;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          clean[d] = vf[d];
          odd |= drop_odd<T>(clean[d]);
        }
        if (__any(odd)) {
#pragma unroll 1
          for (int kind = 0; kind < 3; ++kind)
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              const f32x4 seen = Mma<T>::mul(marks<T>(vf[d], kind), p, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (seen[i] > 0.0f) o[d][i] += marked(kind);
            }
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) vf[d] = clean[d];
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] = Mma<T>::mul(vf[d], p, o[d]);
    }
  }
  w.mx = mx;
  w.sum = sum;
}

// The `waves` of an item, this one of them being number wk, join in halves through LDS (32 outputs, m and
// l of a lane); the first of them writes the item's part.
template <typename T>
__device__ inline void stream_end(StreamState<T>& w, const SharedArgs& a, const Item& it, int wave, int waves,
                                  float* lds) {
  const int lane = threadIdx.x & 63, g = lane >> 4, wk = wave & (waves - 1);
  f32x4 (&o)[8] = w.o;
  float mx = w.mx, sum = over_groups_sum(w.sum, 16);
  for (int half = waves >> 1; half > 0; half >>= 1) {
    float* at = lds + (wave / waves * (waves >> 1) + (wk & (half - 1))) * 34 * 64 + lane;
    if (wk >= half && wk < 2 * half) {
#pragma unroll
      for (int e = 0; e < 32; ++e) at[e * 64] = o[e >> 2][e & 3];
      at[32 * 64] = mx;
      at[33 * 64] = sum;
    }
    __syncthreads();
    if (wk < half) {
      const float m2 = at[32 * 64], l2 = at[33 * 64];
      const float top = fmaxf(mx, m2), ms = top == -INFINITY ? 0.0f : top;
      const float x = __builtin_amdgcn_exp2f(mx - ms), y = __builtin_amdgcn_exp2f(m2 - ms);
      mx = top;
      sum = sum * x + l2 * y;
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e >> 2][e & 3] = o[e >> 2][e & 3] * x + at[e * 64] * y;
    }
    __syncthreads();
  }
  if (wk > 0 || w.m >= it.m1) return;
  T* dst = nullptr;
  const float inv = row_out<T>(a, it, w.m, mx, sum, g == 0, &dst);
#pragma unroll
  for (int d = 0; d < 8; ++d) put4<T>(a, it, w.m, 16 * d + 4 * g, o[d], inv, dst);
}

// `waves` of the workgroup (1, 2, 4 or 8, the same for all its items) work on one item.  All waves of the
// workgroup come here: those without an item with m0 == m1.
template <typename T, bool OWN>
__device__ inline void stream_item(const SharedArgs& a, const Source& src, const Item& it, int waves, float* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_page = (src.T + kStep - 1) / kStep, n_steps = steps_of(src, it.n_keys, kStep, per_page);
  const int share = it.n_split * waves, mine = it.split * waves + (wave & (waves - 1));
  StreamState<T> w;
  stream_begin(w, a, it);
  stream_steps<T, OWN>(w, a, src, it, per_page, share_of(n_steps, mine, share), share_of(n_steps, mine + 1, share));
  stream_end(w, a, it, wave, waves, lds);
}

// The only sequence of a call with few rows and keys, one part: the prefix's keys and then its own.
template <typename T>
__device__ inline void stream_both(const SharedArgs& a, const Item& pre, const Item& own, float* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pp = (a.pre.T + kStep - 1) / kStep, po = (a.own.T + kStep - 1) / kStep;
  const int n_pre = steps_of(a.pre, pre.n_keys, kStep, pp), n = n_pre + steps_of(a.own, own.n_keys, kStep, po);
  const int s0 = share_of(n, wave, kWaves), s1 = share_of(n, wave + 1, kWaves);
  StreamState<T> w;
  stream_begin(w, a, own);
  stream_steps<T, false>(w, a, a.pre, pre, pp, s0, s1 < n_pre ? s1 : n_pre);
  stream_steps<T, true>(w, a, a.own, own, po, s0 < n_pre ? 0 : s0 - n_pre, s1 - n_pre);
  stream_end(w, a, own, wave, kWaves, lds);
}

// ---- more rows: waves of 32 rows share tiles of 64 keys in LDS, on 32x32x16 MFMAs ---------------
// K lies in LDS as two halves of 64 channels, 128 B a key, V^T as 128 B (64 keys) a channel; a direct
// global -> LDS load fills 8 such rows, so it reads whole 128 B lines.  16 B piece c of row r holds piece
// c ^ (r / 2) % 8 of the row in memory: the 16 lanes that an operand read serves at once then fall on
// different banks.  Row i of a K operand is key 16 (i / 16) + 8 ((i / 4) % 2) + 4 ((i / 8) % 2) + i % 4
// of its 32: the 16 scores of lane (n, hh) are then row n's keys 8 hh .. 8 hh + 7 and 16 + 8 hh .. + 7.
constexpr int kBlock = 1024;  // bytes that a wave's direct load fills
constexpr int kRing = 4;  // tiles in LDS
constexpr int kTileLds = kRing * 32 * kBlock;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) char lds_char;

// Where a tile lies and what of it exists.
struct TileAt {
  int64_t base;  // elements to its page's rows of the head (K and V alike); page 0 where there is none
  int key0;      // number of its first key
  int tok0;      // its first token in the page
  int valid;     // keys that exist
};

struct TileWalk {
  PageWalk pages;
  int page, in_page, per_page, id;
  __device__ void start(const Item& it, int per, int tile) {
    per_page = per;
    page = tile / per;
    in_page = tile - page * per;
    pages.start(it.list, it.n_list, page);
  }
  __device__ void first() {
    pages.landed();
    id = pages.get(page);
  }
  __device__ void next() {
    if (++in_page == per_page) {
      in_page = 0;
      id = pages.get(++page);
    }
  }
  // head_size: elements of a page's rows of one head
  __device__ TileAt at(const Source& src, const Item& it, int heads, int64_t head_size) const {
    TileAt x;
    const bool there = id >= 0 && id < src.n_pages;
    x.base = ((int64_t)(there ? id : 0) * heads + it.h) * head_size;
    x.tok0 = in_page * kTile;
    x.key0 = page * src.T + x.tok0;
    int left = it.n_keys - x.key0;
    if (left > src.T - x.tok0) left = src.T - x.tok0;
    x.valid = there ? (left > kTile ? kTile : left) : 0;
    return x;
  }
};

// A wave's share of a tile: 8 keys of K and twice 8 channels of V^T.  `lane` and `dst` are its own.
template <typename T>
__device__ inline void stage_k(const Source& src, const TileAt& x, int klane, lds_char* dst, int wave) {
  const T* kt = static_cast<const T*>(src.k_pool) + x.base + x.tok0 * kHeadDim;
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)kt, (short)0, 0x7fffffff, 0x00020000);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(dst + (8 * i + wave) * kBlock), 16, klane,
                                             (8 * wave * kHeadDim + 64 * i) * 2, 0, 0);
}
template <typename T>
__device__ inline void stage_v(const Source& src, const TileAt& x, int vlane, lds_char* dst, int wave) {
  const T* vt = static_cast<const T*>(src.v_pool) + x.base + x.tok0;
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)vt, (short)0, 0x7fffffff, 0x00020000);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(dst + (8 * i + wave) * kBlock), 16, vlane,
                                             8 * (wave + 8 * i) * src.Tp * 2, 0, 0);
}

// Where a load into `at` of LDS goes, as a number that hipcc cannot trace to the array: where it can, it
// waits for every load under way ahead of a round's first read (7 to 14% of a tile's time); the loops
// below count their waits.
__device__ inline lds_char* load_target(char* at) {
  uint32_t to = (uint32_t)(uintptr_t)(lds_char*)at;
  asm volatile("" : "+s"(to));
  return (lds_char*)(uintptr_t)to;
}

// 16 products with their LDS operands read four ahead.
__device__ inline void ahead_of_products() {
  __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
  for (int i = 0; i < 12; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
}

template <typename T>
struct TileState {
  typename Mma<T>::v8 q[8];
  f32x16 o[4];
  float mx, sum;
};

// The probabilities of a tile at the running maximum, without looking for the tile's own: only when a
// lane's sum leaves [0, 2^8] (or the row has no maximum yet) does the wave take the true maximum,
// rescale what it has and form the tile's probabilities again.
template <typename T>
__device__ inline float probs(const f32x16 (&sc)[2], float c, float mx, typename Mma<T>::v8 (&p)[4]) {
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float e = __builtin_amdgcn_exp2f(sc[i >> 4][i & 15] * c - mx);
    sum += e;
    p[i >> 3][i & 7] = (T)e;  // rounded to the pool's type; the sum is of fp32 values
  }
  return sum;
}

template <typename T>
__device__ inline void settle(TileState<T>& w, const f32x16 (&sc)[2], float c, float sum, typename Mma<T>::v8 (&p)[4],
                              bool odd) {
  if (__any(odd)) {
    float top = sc[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, sc[i >> 4][i & 15]);
    top = over_groups_max(top, 32) * c;
    const float m2 = fmaxf(w.mx, top);
    const float f = m2 == w.mx ? 1.0f : __builtin_amdgcn_exp2f(w.mx - m2);
    w.mx = m2;
    w.sum *= f;
#pragma unroll
    for (int d = 0; d < 4; ++d) w.o[d] *= f;
    sum = probs<T>(sc, c, m2 == -INFINITY ? 0.0f : m2, p);
  }
  w.sum += sum;
}

// Scores of keys `most` and beyond (of a lane's 32: register i is key 16 (i / 8) + i % 8) become -infinity.
// A compare and a choice each: as plain code hipcc makes all 32 comparisons first and spills them.
template <int KEY>
__device__ inline float unless_seen(float x, int most, float none) {
  asm("v_cmp_lt_i32 vcc, %2, %1\n\tv_cndmask_b32 %0, %3, %0, vcc" : "+v"(x) : "v"(most), "n"(KEY), "v"(none) : "vcc");
  return x;
}
template <int KK, int... I>
__device__ inline void mask_eight(f32x16& sc, int most, std::integer_sequence<int, I...>) {
  const float none = -INFINITY;
  ((sc[8 * (KK & 1) + I] = unless_seen<16 * KK + I>(sc[8 * (KK & 1) + I], most, none)), ...);
}
// `from`: keys below it need no look, the same for the whole wave
template <int... KK>
__device__ inline void mask_keys(f32x16 (&sc)[2], int most, int from, std::integer_sequence<int, KK...>) {
  ((16 * KK + 16 > from ? mask_eight<KK>(sc[KK >> 1], most, std::make_integer_sequence<int, 8>{}) : void()), ...);
}

// The second product of a tile that has keys which do not exist, or (OWN) that some rows do not see.
template <typename T, bool OWN>
__device__ inline void masked_pv(TileState<T>& w, const TileAt& x, bool partial, const char* vt,
                                 const int (&piece)[4], const typename Mma<T>::v8 (&p)[4]) {
  typedef typename Mma<T>::v8 v8;
  const int hh = (threadIdx.x & 63) >> 5;
  bool odd = false;
  v8 v[4], ahead[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) v[d] = *reinterpret_cast<const v8*>(vt + piece[0] + d * 4 * kBlock);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (16 * kk >= x.valid) break;
    if (kk < 3 && 16 * kk + 16 < x.valid) {
#pragma unroll
      for (int d = 0; d < 4; ++d) ahead[d] = *reinterpret_cast<const v8*>(vt + piece[kk + 1] + d * 4 * kBlock);
    }
    if (16 * kk + 16 > x.valid) {
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] = drop_behind(v[d], 16 * kk + 8 * hh, x.valid);
    }
    if (partial) {  // as in stream_item
#pragma unroll
      for (int d = 0; d < 4; ++d) odd |= drop_odd<T>(v[d]);
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) w.o[d] = Mma<T>::mul(v[d], p[kk], w.o[d]);
#pragma unroll
    for (int d = 0; d < 4; ++d) v[d] = ahead[d];
  }
  // The products' results are copied on some of the paths from here, which hipcc has left short of their
  // wait states: they wait here.
  asm volatile("s_nop 11" : "+v"(w.o[0]), "+v"(w.o[1]), "+v"(w.o[2]), "+v"(w.o[3]));
  if (OWN && __any(odd)) {
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        f32x16 seen;
#pragma unroll
        for (int i = 0; i < 16; ++i) seen[i] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const v8 raw = *reinterpret_cast<const v8*>(vt + piece[kk] + d * 4 * kBlock);
          seen = Mma<T>::mul(marks<T>(drop_behind(raw, 16 * kk + 8 * hh, x.valid), kind), p[kk], seen);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (seen[i] > 0.0f) w.o[d][i] += marked(kind);
      }
  }
}

// Queries and an empty state of row m, and where a lane's loads and operand reads lie.
template <typename T>
__device__ inline void tile_begin(TileState<T>& w, const SharedArgs& a, const Item& it, int m, int hh) {
  int b, l, gh;
  row_of(a, m, b, l, gh);
  const T* p = static_cast<const T*>(a.q) + b * a.q_sb + l * a.q_st +
               (int64_t)(it.h * a.group + gh) * a.q_sh + hh * 8;
#pragma unroll
  for (int st = 0; st < 8; ++st) w.q[st] = *reinterpret_cast<const typename Mma<T>::v8*>(p + st * 16);
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[d][i] = 0.0f;
  w.mx = -INFINITY;
  w.sum = 0.0f;
}
__device__ inline void tile_lanes(const Source& src, int wave, int lane, int& klane, int& vlane, int (&kpiece)[4],
                                  int (&vpiece)[4]) {
  const int n = lane & 31, hh = lane >> 5, key_row = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
  // loads: lane (r, c) of a wave takes row r of its 8, piece c ^ (row / 2) % 8
  const int from = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
  klane = ((lane >> 3) * kHeadDim + from * 8) * 2;
  vlane = ((lane >> 3) * src.Tp + from * 8) * 2;
  // operand reads: where pieces 2 i + hh of the lane's K row and V^T row lie
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    kpiece[i] = key_row * 128 + (((2 * i + hh) ^ ((key_row >> 1) & 7)) * 16);
    vpiece[i] = n * 128 + (((2 * i + hh) ^ ((n >> 1) & 7)) * 16);
  }
}

// Row m's part, or its output.
template <typename T>
__device__ inline void tile_end(const TileState<T>& w, const SharedArgs& a, const Item& it, int m, bool mine, int hh,
                                float sum) {
  if (!mine) return;
  T* dst = nullptr;
  const float inv = row_out<T>(a, it, m, w.mx, sum, hh == 0, &dst);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = w.o[i >> 2][4 * (i & 3) + e];
    put4<T>(a, it, m, 32 * (i >> 2) + 8 * (i & 3) + 4 * hh, x, inv, dst);
  }
}

// Values of a tile's V^T in LDS at keys `valid` and beyond become zero: all threads, four a channel.
template <typename T>
__device__ inline void drop_keys(char* vt, int valid) {
  typedef typename Mma<T>::v8 v8;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // nothing of this is worth registers in the loop around it
  const int r = tid >> 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = 2 * (tid & 3) + i, k0 = 8 * (c ^ ((r >> 1) & 7));
    v8* const at = reinterpret_cast<v8*>(vt + r * 128 + c * 16);
    if (k0 >= valid) *at = __builtin_bit_cast(v8, u32x4{0u, 0u, 0u, 0u});
    else if (k0 + 8 > valid) *at = drop_behind(*at, k0, valid);
  }
}

// 256 rows against n_own tiles of keys that all of them see as far as they exist, software-pipelined: round t
// holds the scores of tile t + 1, the probabilities of tile t and the second product of tile t - 1, 32
// products with a slice of the softmax after each, so that the matrix cores and the vector units work at the
// same time (753 -> 700 us for 1024 rows of 8 heads against 131072 keys and own pages; one after the other,
// with only the other wave of a SIMD to overlap, before).  K and V have rings of their own: K t + 1 and V t - 1
// are in use while K t + 2 .. t + 4 and V t .. t + 2 are on their way.  kw and vw have started at tile 0.
template <typename T>
__device__ inline __attribute__((always_inline)) void open_tiles(TileState<T>& w, TileWalk& kw, TileWalk& vw, const SharedArgs& a, const Source& src,
                                  const Item& it, int n_own, bool busy, int wave, int klane, int vlane,
                                  const int (&kpiece)[4], const int (&vpiece)[4], char* lds) {
  typedef typename Mma<T>::v8 v8;
  const int64_t head_size = (int64_t)src.Tp * kHeadDim;
  char* const vlds = lds + kRing * 16 * kBlock;
  int valid[kRing];  // keys of tiles t .. t + 3 at round t
  auto load_k = [&](int t) __attribute__((always_inline)) {
    if (t == 0) kw.first();
    else kw.next();
    const TileAt x = kw.at(src, it, a.heads, head_size);
    stage_k<T>(src, x, klane, load_target(lds + (t & (kRing - 1)) * 16 * kBlock), wave);
    return x.valid;
  };
  auto load_v = [&](int t) __attribute__((always_inline)) {
    if (t == 0) vw.first();
    else vw.next();
    stage_v<T>(src, vw.at(src, it, a.heads, head_size), vlane, load_target(vlds + (t & (kRing - 1)) * 16 * kBlock), wave);
  };
  // round 0 multiplies the tile in front of the first by nothing
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *reinterpret_cast<u32x4*>(vlds + (kRing - 1) * 16 * kBlock + (threadIdx.x + i * 64 * kWaves) * 16) = u32x4{0u, 0u, 0u, 0u};
  // The queries' own wait, ahead of the counted ones: they left with the page list, without which no key loads.
#pragma unroll
  for (int st = 0; st < 8; ++st) asm volatile("" : "+v"(w.q[st]));
  if (n_own >= kRing) {
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      valid[i] = load_k(i);
      if (i >= 2) load_v(i - 2);
    }
    asm volatile("s_waitcnt vmcnt(10) lgkmcnt(0)" ::: "memory");  // K 0; the other ten loads may be under way
  } else {
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      valid[i] = kTile;
      if (i < n_own) valid[i] = load_k(i);
      if (i >= 2 && i - 2 < n_own) load_v(i - 2);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }
  auto mask = [&](f32x16 (&sc)[2], int keys) __attribute__((always_inline)) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // keeps this a branch: most tiles have nothing to mask
    const int most = keys - ((tid & 32) >> 2);
    mask_keys(sc, most, keys, std::make_integer_sequence<int, 4>{});
  };
  f32x16 sa[2], sb[2], zero;
  v8 pa[4], pb[4];
#pragma unroll
  for (int i = 0; i < 16; ++i) zero[i] = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) pa[i][e] = (T)0.0f;
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (busy) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      sa[i & 1] = Mma<T>::mul(*reinterpret_cast<const v8*>(lds + kpiece[(i >> 1) & 3] + ((i >> 3) * 8 + (i & 1) * 4) * kBlock),
                              w.q[i >> 1], i < 2 ? zero : sa[i & 1]);
    if (valid[0] < kTile) mask(sa, valid[0]);
    float top = sa[0][0];  // the running maximum starts at the first tile's
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, sa[i >> 4][i & 15]);
    w.mx = over_groups_max(top, 32) * a.c;
  }
  auto round = [&](int t, f32x16 (&cur)[2], f32x16 (&nxt)[2], v8 (&pprev)[4], v8 (&p)[4]) __attribute__((always_inline)) {
    // K t + 1 and V t - 1 have landed (a wave's loads land in order; what was issued behind them may be
    // under way), and everybody is done with K t and V t - 2, whose places load next
    const bool cut = valid[0] < kTile;  // tile t, the same for all waves: V t too, to lose what is no key
    if (t + 3 < n_own) {
      if (cut) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else if (cut || t + 1 >= n_own) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (cut) drop_keys<T>(vlds + (t & (kRing - 1)) * 16 * kBlock, valid[0]);
    const char* const vt = vlds + ((t - 1) & (kRing - 1)) * 16 * kBlock;
    const char* const kt = lds + ((t + 1) & (kRing - 1)) * 16 * kBlock;
    const int next_valid = valid[1];
#pragma unroll
    for (int i = 0; i + 1 < kRing; ++i) valid[i] = valid[i + 1];
    if (t + kRing < n_own) valid[kRing - 1] = load_k(t + kRing);
    if (t + 2 < n_own) load_v(t + 2);
    if (!busy) return;
    // product i: even ones score, odd ones add values
    auto operand = [&](int i) __attribute__((always_inline)) {
      const int st = i >> 1;
      return (i & 1) == 0 ? *reinterpret_cast<const v8*>(kt + kpiece[(st >> 1) & 3] + ((st >> 3) * 8 + (st & 1) * 4) * kBlock)
                          : *reinterpret_cast<const v8*>(vt + vpiece[st >> 2] + (st & 3) * 4 * kBlock);
    };
    v8 ahead[4];
#pragma unroll
    for (int i = 0; i < 3; ++i) ahead[i] = operand(i);
    const float ms = w.mx == -INFINITY ? 0.0f : w.mx;
    float e[32], part[4], sum = 0.0f;
    bool odd = false;
    auto expo = [&](int i) __attribute__((always_inline)) {
      e[i] = __builtin_amdgcn_exp2f(cur[i >> 4][i & 15] * a.c - ms);
      asm volatile("" ::"v"(e[i]));  // stays behind its product
    };
    auto retire = [&](int i) __attribute__((always_inline)) {
      part[i & 3] = i < 4 ? e[i] : part[i & 3] + e[i];
      asm volatile("" ::"v"(part[i & 3]));
      p[i >> 3][i & 7] = (T)e[i];  // rounded to the pool's type; the sum is of fp32 values
      if ((i & 7) == 7) asm volatile("" ::"v"(p[i >> 3]));
    };
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i + 3 < 32) ahead[(i + 3) & 3] = operand(i + 3);
      if (i == 0) __builtin_amdgcn_s_setprio(2);
      if (i == 11) __builtin_amdgcn_s_setprio(1);
      if (i == 22) __builtin_amdgcn_s_setprio(0);
      const int st = i >> 1;
      if ((i & 1) == 0) nxt[st & 1] = Mma<T>::mul(ahead[i & 3], w.q[st >> 1], st < 2 ? zero : nxt[st & 1]);
      else w.o[st & 3] = Mma<T>::mul(ahead[i & 3], pprev[st >> 2], w.o[st & 3]);
      // two probabilities after each of the first products, one after the others; a probability is
      // summed and packed a product later than it is formed
      if (i >= 1 && i <= 4) {
        retire(2 * (i - 1));
        retire(2 * (i - 1) + 1);
      } else if (i >= 5 && i <= 28) {
        retire(i + 3);
      }
      if (i < 4) {
        expo(2 * i);
        expo(2 * i + 1);
      } else if (i < 28) {
        expo(i + 4);
      }
      if (i == 30) {
        sum = (part[0] + part[1]) + (part[2] + part[3]);
        odd = !(sum <= 256.0f) || w.mx == -INFINITY;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    settle<T>(w, cur, a.c, sum, p, odd);
    if (t + 1 < n_own && next_valid < kTile) mask(nxt, next_valid);
  };
  int t = 0;
  for (; t + 1 < n_own; t += 2) {
    round(t, sa, sb, pa, pb);
    round(t + 1, sb, sa, pb, pa);
  }
  if (t < n_own) round(t, sa, sb, pa, pb);
  const int last = n_own - 1;
  const char* const vt = vlds + (last & (kRing - 1)) * 16 * kBlock;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (busy) {  // the last tile's second product
#pragma unroll
    for (int i = 0; i < 16; ++i)
      w.o[i & 3] = Mma<T>::mul(*reinterpret_cast<const v8*>(vt + vpiece[i >> 2] + (i & 3) * 4 * kBlock),
                               n_own & 1 ? pb[i >> 2] : pa[i >> 2], w.o[i & 3]);
  }
}

// An item of 256 rows (WK = 1), or of 128 rows against two tiles a round (WK = 2: waves 0..3 work on the
// first and waves 4..7 on the second).  256 rows take the tiles that all of them see whole as above;
// what is left, and 128 rows, go tile by tile with the masks of their rows.
template <typename T, int WK, bool OWN>
__device__ inline void tile_item(const SharedArgs& a, const Source& src, const Item& it, char* lds) {
  typedef typename Mma<T>::v8 v8;
  constexpr int kRows = kWaves / WK;  // waves side by side
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hh = lane >> 5, wr = wave % kRows, wk = wave / kRows;
  const int per_page = (src.T + kTile - 1) / kTile;
  const int n_tiles = steps_of(src, it.n_keys, kTile, per_page);
  const int t0 = share_of(n_tiles, it.split, it.n_split), n_own = share_of(n_tiles, it.split + 1, it.n_split) - t0;
  // the tiles that go ahead of the others; a few are not worth the start
  int n_open = 0;
  if constexpr (WK == 1) {
    const int whole = it.open >= it.n_keys ? n_tiles : it.open / src.T * per_page + it.open % src.T / kTile;
    n_open = whole - t0 < n_own ? whole - t0 : n_own;
    if (OWN && n_open < 4) n_open = 0;
  }
  TileWalk walk, ahead;  // at the tile that loads last
  if (n_own > 0) {       // the page lists load while the rows are looked up
    walk.start(it, per_page, t0);
    if (WK == 1) ahead.start(it, per_page, t0);
  }
  const bool busy = it.m0 + 32 * wr < it.m1;  // the wave has rows at all
  const bool mine = it.m0 + 32 * wr + n < it.m1;
  const int m = all_rows(a, it, mine ? it.m0 + 32 * wr + n : it.m0);
  int b, l, gh;
  row_of(a, m, b, l, gh);
  const int lim = OWN ? keys_seen(it, l) : it.n_keys;
  TileState<T> w;
  tile_begin(w, a, it, m, hh);
  int klane, vlane, kpiece[4], vpiece[4];
  tile_lanes(src, wave, lane, klane, vlane, kpiece, vpiece);
  if constexpr (WK == 1) {
    if (n_open > 0) {
      open_tiles<T>(w, ahead, walk, a, src, it, n_open, busy, wave, klane, vlane, kpiece, vpiece, lds);
      if (n_open < n_own) {
        walk.start(it, per_page, t0 + n_open);
        __builtin_amdgcn_s_barrier();  // everybody is done with what lies in LDS
        asm volatile("" ::: "memory");
      }
    }
  }
  const int n_rest = WK == 2 || OWN ? n_own - n_open : 0;
  const int64_t head_size = (int64_t)src.Tp * kHeadDim;
  TileAt ring[kRing - WK];  // the tiles in use and those on their way
  auto stage = [&](TileAt& x, int t) {
    if (t == 0) walk.first();
    else walk.next();
    x = walk.at(src, it, a.heads, head_size);
    lds_char* const to = load_target(lds + (t & (kRing - 1)) * 32 * kBlock);
    stage_k<T>(src, x, klane, to, wave);
    stage_v<T>(src, x, vlane, to + 16 * kBlock, wave);
  };
#pragma unroll
  for (int i = 0; i < kRing - WK; ++i) {
    ring[i] = TileAt{};
    if (i < n_rest) stage(ring[i], i);
  }
  // the queries' own wait, ahead of the loop's counted ones
#pragma unroll
  for (int st = 0; st < 8; ++st) asm volatile("" : "+v"(w.q[st]));
  for (int t = 0; t < n_rest; t += WK) {
    // This round's tiles have landed (a wave's loads land in order: what was issued after them may
    // still be under way), and everybody is done with the round before, whose buffers load next.
    constexpr int kLoads = 4;  // of a wave and tile
    if (WK == 1 && t + 2 < n_rest) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
    else if (WK == 1 && t + 1 < n_rest) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const TileAt cur = WK == 2 && wk == 1 ? ring[1] : ring[0];
#pragma unroll
    for (int i = 0; i + WK < kRing - WK; ++i) ring[i] = ring[i + WK];
#pragma unroll
    for (int i = 0; i < WK; ++i)
      if (t + kRing - WK + i < n_rest) stage(ring[kRing - 2 * WK + i], t + kRing - WK + i);
    const char* const kt = lds + ((t + wk) & (kRing - 1)) * 32 * kBlock;
    const char* const vt = kt + 16 * kBlock;
    if (busy && t + wk < n_rest) {
      f32x16 sc[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[0][i] = sc[1][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sc[i & 1] = Mma<T>::mul(*reinterpret_cast<const v8*>(kt + kpiece[(i >> 1) & 3] + ((i >> 3) * 8 + (i & 1) * 4) * kBlock),
                                w.q[i >> 1], sc[i & 1]);
      ahead_of_products();
      const bool partial = OWN && cur.key0 + cur.valid > it.open, masked = cur.valid < kTile || partial;
      if (masked) {
        const int seen = lim - cur.key0;
        int most = (seen < cur.valid ? seen : cur.valid) - 8 * hh;
        asm volatile("" : "+v"(most));  // keeps this a branch: most tiles have nothing to mask
        mask_keys(sc, most, OWN ? 0 : cur.valid, std::make_integer_sequence<int, 4>{});
      }
      v8 p[4];
      const float sum = probs<T>(sc, a.c, w.mx == -INFINITY ? 0.0f : w.mx, p);
      settle<T>(w, sc, a.c, sum, p, !(sum <= 256.0f) || w.mx == -INFINITY);
      if (masked) {
        masked_pv<T, OWN>(w, cur, partial, vt, vpiece, p);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w.o[i & 3] = Mma<T>::mul(*reinterpret_cast<const v8*>(vt + vpiece[i >> 2] + (i & 3) * 4 * kBlock), p[i >> 2],
                                   w.o[i & 3]);
        ahead_of_products();
      }
    }
  }
  float sum = over_groups_sum(w.sum, 32);
  if constexpr (WK == 2) {  // the two halves of the waves join through LDS
    float* const at = reinterpret_cast<float*>(lds) + wr * 66 * 64 + lane;
    __syncthreads();
    if (wk == 1) {
#pragma unroll
      for (int i = 0; i < 64; ++i) at[i * 64] = w.o[i >> 4][i & 15];
      at[64 * 64] = w.mx;
      at[65 * 64] = sum;
    }
    __syncthreads();
    if (wk == 1) return;
    const float m2 = at[64 * 64], l2 = at[65 * 64];
    const float top = fmaxf(w.mx, m2), ms = top == -INFINITY ? 0.0f : top;
    const float x = __builtin_amdgcn_exp2f(w.mx - ms), y = __builtin_amdgcn_exp2f(m2 - ms);
    w.mx = top;
    sum = sum * x + l2 * y;
#pragma unroll
    for (int i = 0; i < 64; ++i) w.o[i >> 4][i & 15] = w.o[i >> 4][i & 15] * x + at[i * 64] * y;
  }
  tile_end(w, a, it, m, mine, hh, sum);
}


__device__ inline void prefix_keys(const SharedArgs& a, Item& it) {
  it.list = a.pre_pages;
  it.n_list = (int)((a.pre_tokens + a.pre.T - 1) / a.pre.T);
  it.n_keys = it.open = (int)a.pre_tokens;
  it.first_lim = 0;
  it.causal = false;
}

// The keys of sequence b that rows [m0, m1) see; `none`: there is no item.
__device__ inline void own_keys(const SharedArgs& a, Item& it, int b, bool none) {
  const int per = a.rows * a.group;
  it.tokens = nullptr;
  it.list = a.tables + b * a.table_st;
  it.n_list = a.width;
  it.causal = a.causal;
  // row l of a causal sequence sees lengths - fresh + l + 1 keys; keys past the table do not exist
  const int fresh = fresh_rows(a, b), l0 = (it.m0 - b * per) / a.group, l1 = (it.m1 - 1 - b * per) / a.group;
  const int64_t length = a.lengths[b], cap = (int64_t)a.width * a.own.T;
  it.first_lim = length - fresh + 1;
  int64_t keys = a.causal && it.first_lim + l1 < length ? it.first_lim + l1 : length;
  if (keys > cap) keys = cap;
  if (keys < 0 || l0 >= fresh || none) keys = 0;  // no row of the item is a new token
  it.n_keys = (int)keys;
  it.open = !a.causal ? it.n_keys : it.first_lim + l0 < 0 ? 0 : it.first_lim + l0 < keys ? (int)it.first_lim + l0 : it.n_keys;
}

// The prefix's work items first, dealt so that the row blocks of one (key head, split) run one after
// another on one XCD and share its L2 (interleaved with the others 765 -> 947 us at 1024 rows of 8 heads
// against 131072 keys); then every sequence's own pages.  PK, OK: how the prefix and the
// own pages go (0: streaming, else tiles a round).
template <typename T, int PK, int OK>
__global__ __launch_bounds__(64 * kWaves, 2) void attend_shared_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[PK || OK ? kTileLds : kWaves / 2 * 34 * 64 * 4];
  __shared__ int tokens[PK ? kCompact + 1 : 1];
  Item it;
  if constexpr (PK == 0 && OK == 0) {
    if (a.both) {
      Item pre;
      it.h = pre.h = blockIdx.x;
      it.part = 0;
      it.m0 = 0;
      it.m1 = a.M;
      prefix_keys(a, pre);
      own_keys(a, it, 0, false);
      stream_both<T>(a, pre, it, reinterpret_cast<float*>(lds));
      return;
    }
  }
  if ((int)blockIdx.x < a.pre_grid) {
    constexpr int R = kind_rows(PK);
    int rows = a.M;
    it.tokens = nullptr;
    if constexpr (PK) {
      // a padded batch: its new tokens close up, so that the prefix meets rows that count
      if (a.new_lens != nullptr && a.batch <= kCompact && !a.direct) {
        if (threadIdx.x < 64) {
          int sum = 0;
          for (int b0 = 0; b0 < a.batch; b0 += 64) {
            const int i = b0 + threadIdx.x, n = i < a.batch ? fresh_rows(a, i) : 0;
            int upto = n;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
              const int other = __shfl_up(upto, d, 64);
              if ((int)threadIdx.x >= d) upto += other;
            }
            if (i < a.batch) tokens[i] = sum + upto - n;
            sum += __shfl(upto, 63, 64);
          }
          if (threadIdx.x == 0) tokens[a.batch] = sum;
        }
        __syncthreads();
        it.tokens = tokens;
        rows = __builtin_amdgcn_readfirstlane(tokens[a.batch]) * a.group;
      }
    }
    // every eighth workgroup runs on the same XCD: each gets an equal run of (key head, split)s' row blocks
    const int blocks = (rows + R - 1) / R, n = a.heads * a.pre_splits * blocks, each = (n + 7) / 8;
    const int at = blockIdx.x >> 3, unit = (blockIdx.x & 7) * each + at;
    if (at >= each || unit >= n) return;
    const int pair = unit / blocks;
    it.h = pair % a.heads;
    it.split = it.part = pair / a.heads;
    it.n_split = a.pre_splits;
    it.m0 = (unit - pair * blocks) * R;
    it.m1 = it.m0 + R < rows ? it.m0 + R : rows;
    prefix_keys(a, it);
    if constexpr (PK) tile_item<T, PK, false>(a, a.pre, it, lds);
    else stream_item<T, false>(a, a.pre, it, kWaves, reinterpret_cast<float*>(lds));
    return;
  }
  constexpr int R = kind_rows(OK);
  // a workgroup that streams takes as many items as its waves make
  const int waves = OK ? kWaves : a.own_waves;
  int bid = ((int)blockIdx.x - a.pre_grid) * (kWaves / waves) +
            __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / waves;
  const bool none = bid >= a.own_items;
  if (none) bid = 0;
  it.split = bid % a.own_splits;
  bid /= a.own_splits;
  const int rb = bid % a.own_rb;
  bid /= a.own_rb;
  it.h = bid % a.heads;
  const int b = bid / a.heads, per = a.rows * a.group;
  it.n_split = a.own_splits;
  it.part = a.pre_splits + it.split;
  it.m0 = b * per + rb * R;
  it.m1 = it.m0 + R < (b + 1) * per ? it.m0 + R : (b + 1) * per;
  if (none) it.m1 = it.m0;
  own_keys(a, it, b, none);
  if constexpr (OK) tile_item<T, OK, true>(a, a.own, it, lds);
  else stream_item<T, true>(a, a.own, it, waves, reinterpret_cast<float*>(lds));
}

// The join of up to kFewParts parts: half a wave per (row, key head), a lane four channels, all parts'
// values under way at once (3 parts of 18720 rows, 29 MB, 7.6 us; a wave a row as below 13.3).
constexpr int kFewParts = 8;
template <typename T>
__global__ __launch_bounds__(256) void merge_few_kernel(SharedArgs a, int n_parts) {
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int c = 4 * (threadIdx.x & 31);
  if (unit >= (int64_t)a.heads * a.M) return;
  const int h = (int)(unit % a.heads), m = (int)(unit / a.heads);
  int b, l, gh;
  row_of(a, m, b, l, gh);
  const int64_t at = (int64_t)h * a.M + m, step = (int64_t)a.heads * a.M;
  f32x4 v[kFewParts], o = f32x4{0.f, 0.f, 0.f, 0.f};
  float2 ml[kFewParts];
#pragma unroll
  for (int p = 0; p < kFewParts; ++p) {
    if (p >= n_parts) break;
    ml[p] = a.part_ml[at + p * step];
    v[p] = *reinterpret_cast<const f32x4*>(a.part_o + (at + p * step) * kHeadDim + c);
  }
  float top = -INFINITY, total = 0.0f;
#pragma unroll
  for (int p = 0; p < kFewParts; ++p)
    if (p < n_parts) top = fmaxf(top, ml[p].x);
  if (top == -INFINITY) top = 0.0f;
#pragma unroll
  for (int p = 0; p < kFewParts; ++p)
    if (p < n_parts) {
      const float x = __builtin_amdgcn_exp2f(ml[p].x - top);
      total += x * ml[p].y;
      o += x * v[p];
    }
  const bool any = l < fresh_rows(a, b) && total != 0.0f;  // a row that sees no key is zero (NaN sums are not zero)
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = any ? (T)(o[i] / total) : (T)0.0f;
  *reinterpret_cast<t4*>(static_cast<T*>(a.out) + b * a.o_sb + l * a.o_st + (int64_t)(h * a.group + gh) * a.o_sh + c) = r;
}

// One wave per (row, key head).  Lane p weighs part p (64 parts at a time); then each half of the wave
// adds every other part, a lane four channels, with four loads in flight (17 parts of 1024 rows 6.4 us).
template <typename T>
__global__ __launch_bounds__(256) void merge_kernel(SharedArgs a, int n_parts) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, half = lane >> 5, c = 4 * (lane & 31);
  if (unit >= (int64_t)a.heads * a.M) return;
  const int h = (int)(unit % a.heads), m = (int)(unit / a.heads);
  int b, l, gh;
  row_of(a, m, b, l, gh);
  const int64_t at = (int64_t)h * a.M + m, step = (int64_t)a.heads * a.M;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  float total = 0.0f;
  if (l < fresh_rows(a, b)) {
    float top = -INFINITY;
    for (int p = lane; p < n_parts; p += 64) top = fmaxf(top, a.part_ml[at + p * step].x);
    top = over_groups_max(top, 1);
    if (top == -INFINITY) top = 0.0f;
    for (int p0 = 0; p0 < n_parts; p0 += 64) {
      const int n = n_parts - p0 < 64 ? n_parts - p0 : 64;
      float w = 0.0f;
      if (lane < n) {
        const float2 ml = a.part_ml[at + (p0 + lane) * step];
        w = __builtin_amdgcn_exp2f(ml.x - top);
        total += w * ml.y;
      }
      const float* part = a.part_o + (at + p0 * step) * kHeadDim + c;
      // all lanes make every round (a lane that left could not be asked for its weight)
#pragma unroll 1
      for (int p = 0; p < n; p += 8) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int mine = p + i + half;
          const float x = __shfl(w, mine & 63, 64);
          const f32x4 v = *reinterpret_cast<const f32x4*>(part + (mine < n ? mine : 0) * step * kHeadDim);
          if (mine < n) o += x * v;
        }
      }
    }
    total = over_groups_sum(total, 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], 32, 64);
  }
  const bool any = total != 0.0f;  // a row that sees no key is zero (NaN sums are not zero)
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = any ? (T)(o[i] / total) : (T)0.0f;
  T* dst = static_cast<T*>(a.out) + b * a.o_sb + l * a.o_st + (int64_t)(h * a.group + gh) * a.o_sh;
  if (half == 0) *reinterpret_cast<t4*>(dst + c) = r;
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
bool half_dtype(int t) { return t == SKV_BF16 || t == SKV_F16; }

bool view_ok(const void* p, int64_t sb, int64_t st, int64_t sh) {
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb >= 0 && st >= 0 && sh >= 0 &&
         sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0;
}

bool pool_ok(const void* k, const void* v) {
  return k && v && reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0;
}

int launched(const char* fn) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return SKV_OK;
  set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
  return SKV_E_LAUNCH;
}

int common_errors(const char* fn, int dtype, int head_dim, int batch, int rows, int q_heads,
                  int kv_heads, int n_pages, int page_tokens, const int32_t* tables,
                  int64_t table_stride, int table_width, const int32_t* lengths, bool q_needed) {
  if (head_dim != kHeadDim) {
    set_error("%s: head_dim=%d unsupported (built for %d)", fn, head_dim, kHeadDim);
    return SKV_E_UNSUPPORTED;
  }
  if (!half_dtype(dtype)) {
    set_error("%s: dtype %d unsupported (bf16 or f16)", fn, dtype);
    return SKV_E_UNSUPPORTED;
  }
  if (batch < 0 || rows < 0 || kv_heads <= 0 || (q_needed && (q_heads <= 0 || q_heads % kv_heads))) {
    set_error("%s: bad sizes (batch=%d rows=%d, %d query heads over %d key heads)", fn, batch, rows,
              q_heads, kv_heads);
    return SKV_E_ARG;
  }
  if ((int64_t)batch * rows >= ((int64_t)1 << 31)) {
    set_error("%s: too many rows (batch=%d rows=%d)", fn, batch, rows);
    return SKV_E_ARG;
  }
  if (n_pages <= 0 || page_tokens <= 0 || page_tokens > (1 << 20)) {
    set_error("%s: bad pool (%d pages of %d tokens)", fn, n_pages, page_tokens);
    return SKV_E_ARG;
  }
  if (table_width < 0 || (table_width > 0 && (!tables || table_stride < 0)) || !lengths ||
      (int64_t)table_width * page_tokens >= ((int64_t)1 << 31)) {
    set_error("%s: bad page tables (width=%d) or no lengths", fn, table_width);
    return SKV_E_ARG;
  }
  return SKV_OK;
}

// The launch of an attention: whether each kind of work item goes by tiles, and the splits.
struct SharedPlan {
  int pre_kind, own_kind;
  bool both;  // one sequence with few rows and keys: a head's prefix and own keys in one work item
  int pre_splits, pre_grid, own_rb, own_splits, own_items, own_waves, own_grid, parts;
  int64_t bytes;
};

// Key splits, and waves of a streaming item, by what they are estimated to take (microseconds, as
// measured on MI355X).  A workgroup has a CU to itself, so what counts is rounds of workgroups.  A
// workgroup takes kFixed to start and end (7.5 us with two steps).  A tile against 256 rows takes 1.45 us
// of a prefix and 1.55 of own pages while half of the CUs work, and 2.0 and 2.45 when all do (the clock
// follows the power, and own pages are shared by no one), two tiles against 128 rows 2.3.  A streaming CU reads 38 GB/s (64 keys in 0.86 us),
// and the whole chip 4.6 TB/s.  Several parts cost kMerge and the bytes of their partial results.
void choose_splits(const skv_attend_shared_desc* d, int64_t M, int64_t cu, int64_t pre_items, int64_t pre_tiles,
                   int64_t own_items, int64_t own_tiles, SharedPlan* p) {
  constexpr double kFixed = 7.0, kBytes = 4.6e6, kMerge = 7.0, kTileBytes = 32768.0;
  auto tile_cost = [](int kind, bool own, double busy) {
    const double over = busy < 0.5 ? 0.0 : (busy < 1.0 ? busy : 1.0) - 0.5;
    return kind == 0 ? 0.86 : kind == 2 ? 1.15 : own ? 1.55 + 1.8 * over : 1.45 + 1.1 * over;
  };
  // tables are as wide as their longest sequence gets: the average one holds half of that
  const double mean = 0.5 * own_tiles, longer = 0.75 * own_tiles;
  const double own_bytes = mean * own_items * kTileBytes;
  const double stream = ((double)pre_tiles * d->kv_heads * kTileBytes + own_bytes) / kBytes + kFixed;
  // short sequences share a workgroup where there is more than one a CU: at most 4 steps a wave
  int waves = kWaves;
  if (p->own_kind == 0 && own_items > cu)
    while (waves > 1 && own_tiles <= waves) waves >>= 1;
  double best = 1e30;
  p->pre_splits = pre_tiles > 0, p->own_splits = own_tiles > 0, p->own_waves = waves;
  for (int os = 1; os <= (waves == kWaves && own_tiles > 1 ? 32 : 1); os *= 2) {
    const int64_t n_own = own_tiles ? (own_items * os * waves + kWaves - 1) / kWaves : 0;
    // the prefix's workgroups fill what the own ones leave of a round or two, or a part of a round; or one
    // part each
    for (int f = 0; f < (pre_tiles ? 7 : 1); ++f) {
      int64_t ps = 0;
      if (pre_tiles) {
        const int64_t room = f == 0 ? cu - n_own : f == 1 ? 2 * cu - n_own : f < 6 ? cu * (f - 1) / 4 : 0;
        ps = room / pre_items;
        ps = ps < 1 ? 1 : ps > pre_tiles ? pre_tiles : ps > 256 ? 256 : ps;
      }
      const int64_t n_pre = pre_items * ps, full = n_pre / cu, part = n_pre % cu;
      const double busy = (double)(full ? cu : part) / cu;
      const double dp = ps ? kFixed + (double)((pre_tiles + ps - 1) / ps) * tile_cost(p->pre_kind, false, busy) : 0.0;
      const double dn = kFixed + longer / os * tile_cost(p->own_kind, true, (double)n_own / cu) * kWaves / waves;
      double t;
      if (n_pre + n_own <= cu) {
        t = n_own && dn > dp ? dn : dp;
      } else {
        const double rounds = (double)(full + (part > 0)) * dp;
        const double hidden = part ? (double)(cu - part) * dp / dn : 0.0;  // own workgroups beside the last round
        const double left = n_own > hidden ? n_own - hidden : 0.0;
        double tail = left / cu * dn;
        if (tail < left / (n_own ? n_own : 1) * own_bytes / kBytes) tail = left / n_own * own_bytes / kBytes;
        t = rounds + (left > 0 ? tail + 0.5 * dn : 0.0);
      }
      if (t < stream) t = stream;
      if (ps + os * (own_tiles > 0) > 1) t += kMerge + (double)(ps + os) * M * d->kv_heads * 1040 / kBytes;
      if (t < best) {
        best = t;
        p->pre_splits = (int)ps;
        p->own_splits = own_tiles ? os : 0;
      }
    }
  }
}

int plan_shared(const char* fn, const skv_attend_shared_desc* d, SharedPlan* p) {
  const int group = d->q_heads / d->kv_heads;
  const int64_t M = (int64_t)d->batch * d->rows * group, per = (int64_t)d->rows * group;
  *p = SharedPlan{};
  if (M == 0) return SKV_OK;
  if ((M * d->kv_heads + 3) / 4 * 256 >= kMaxThreads) {
    set_error("%s: too many query rows (batch=%d rows=%d heads=%d)", fn, d->batch, d->rows, d->q_heads);
    return SKV_E_ARG;
  }
  const bool pre = d->prefix_tokens > 0, own = d->table_width > 0;
  p->own_kind = kind_of(per);
  p->pre_kind = pre ? kind_of(M) : p->own_kind;
  const int pre_rows = kind_rows(p->pre_kind), own_rows = kind_rows(p->own_kind);
  const int64_t cu = cu_count();
  auto tiles = [](int64_t tokens, int64_t page) {
    return tokens / page * ((page + kTile - 1) / kTile) + (tokens % page + kTile - 1) / kTile;
  };
  const int64_t pre_tiles = pre ? tiles(d->prefix_tokens, d->prefix_page_tokens) : 0;
  const int64_t own_tiles = own ? tiles((int64_t)d->table_width * d->page_tokens, d->page_tokens) : 0;
  const int64_t pre_rb = pre ? (M + pre_rows - 1) / pre_rows : 0;
  p->own_rb = own ? (int)((per + own_rows - 1) / own_rows) : 0;
  const int64_t pre_items = pre_rb * d->kv_heads;
  const int64_t own_items = (int64_t)p->own_rb * d->kv_heads * d->batch;
  // of a padded batch's row blocks about half hold tokens
  const int64_t busy_rb = d->new_lens && p->pre_kind ? (M / 2 + pre_rows) / pre_rows : pre_rb;
  // A sequence by itself with few rows and keys needs no second part and no merge (12.1 us for 390 + 64
  // keys of 12 heads, and 15.3 in two parts); in several parts its own keys are better off beside the
  // prefix (19.6 us for 8190 + 1560 keys of 8 heads, and 22.3 in one list).
  if (pre && own && d->batch == 1 && p->pre_kind == 0) {
    choose_splits(d, M, cu, pre_items, pre_tiles + own_tiles, 0, 0, p);
    p->both = p->pre_splits == 1;
  }
  if (!p->both)
    choose_splits(d, M, cu, busy_rb < pre_rb ? busy_rb * d->kv_heads : pre_items, pre_tiles, own_items, own_tiles, p);
  p->parts = p->pre_splits + p->own_splits;
  const int64_t each = p->own_kind ? 1 : kWaves / p->own_waves;
  const int64_t pre_grid = (pre_items * p->pre_splits + 7) / 8 * 8, all_own = own_items * p->own_splits;
  if ((pre_grid + (all_own + each - 1) / each) * 64 * kWaves >= kMaxThreads) {
    set_error("%s: too many work items", fn);
    return SKV_E_ARG;
  }
  p->pre_grid = p->both ? d->kv_heads : (int)pre_grid;
  p->own_items = (int)all_own;
  p->own_grid = p->both ? 0 : (int)((all_own + each - 1) / each);
  p->bytes = p->parts > 1 ? (int64_t)p->parts * d->kv_heads * M * (kHeadDim * 4 + 8) : 0;
  return SKV_OK;
}

int check_shared(const char* fn, const skv_attend_shared_desc* d) {
  clear_error();
  if (!d) {
    set_error("%s: null descriptor", fn);
    return SKV_E_ARG;
  }
  const int st = common_errors(fn, d->dtype, d->head_dim, d->batch, d->rows, d->q_heads, d->kv_heads,
                               d->n_pages, d->page_tokens, d->tables, d->table_stride, d->table_width,
                               d->lengths, true);
  if (st != SKV_OK) return st;
  if (!view_ok(d->q, d->q_sb, d->q_st, d->q_sh) || !view_ok(d->out, d->out_sb, d->out_st, d->out_sh)) {
    set_error("%s: q and out must be 16-byte aligned with non-negative strides that are multiples of "
              "8 elements", fn);
    return SKV_E_ARG;
  }
  if (!pool_ok(d->k_pool, d->v_pool)) {
    set_error("%s: pools must be 16-byte aligned", fn);
    return SKV_E_ARG;
  }
  if (d->prefix_tokens < 0 ||
      (d->prefix_tokens > 0 &&
       (!pool_ok(d->prefix_k_pool, d->prefix_v_pool) || !d->prefix_pages || d->prefix_n_pages <= 0 ||
        d->prefix_page_tokens <= 0 || d->prefix_page_tokens > (1 << 20) ||
        d->prefix_tokens >= ((int64_t)1 << 31)))) {
    set_error("%s: bad prefix (%lld tokens in pages of %d)", fn, (long long)d->prefix_tokens,
              d->prefix_page_tokens);
    return SKV_E_ARG;
  }
  if (!(d->softmax_scale > 0.0f) || d->softmax_scale > 3.0e38f) {
    set_error("%s: softmax_scale must be positive and finite", fn);
    return SKV_E_ARG;
  }
  return SKV_OK;
}

template <typename T>
void launch_shared(const SharedArgs& a, const SharedPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.pre_grid + p.own_grid)), block(64 * kWaves);
  auto launch = [&](void (*kernel)(SharedArgs)) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a); };
  if (p.pre_kind == 0) launch(attend_shared_kernel<T, 0, 0>);
  else if (p.pre_kind == 2) p.own_kind == 0 ? launch(attend_shared_kernel<T, 2, 0>) : launch(attend_shared_kernel<T, 2, 2>);
  else if (p.own_kind == 0) launch(attend_shared_kernel<T, 1, 0>);
  else if (p.own_kind == 2) launch(attend_shared_kernel<T, 1, 2>);
  else launch(attend_shared_kernel<T, 1, 1>);
}

template <typename T>
void launch_merge(const SharedArgs& a, int parts, hipStream_t s) {
  const int each = parts <= kFewParts ? 8 : 4;
  const dim3 grid((unsigned)(((int64_t)a.heads * a.M + each - 1) / each)), block(256);
  if (parts <= kFewParts) hipLaunchKernelGGL(merge_few_kernel<T>, grid, block, 0, s, a, parts);
  else hipLaunchKernelGGL(merge_kernel<T>, grid, block, 0, s, a, parts);
}

}  // namespace

}  // namespace skv

using namespace skv;

extern "C" int skv_append_pages(const skv_append_pages_desc* d, skv_stream_t stream) {
  const char* fn = "skv_append_pages";
  clear_error();
  if (!d) {
    set_error("%s: null descriptor", fn);
    return SKV_E_ARG;
  }
  int st = common_errors(fn, d->dtype, d->head_dim, d->batch, d->rows, d->q_heads, d->kv_heads, d->n_pages,
                         d->page_tokens, d->tables, d->table_stride, d->table_width, d->lengths, false);
  if (st != SKV_OK) return st;
  const bool q = d->q_heads > 0;
  if (d->q_heads < 0 || !view_ok(d->k, d->k_sb, d->k_st, d->k_sh) || !view_ok(d->v, d->v_sb, d->v_st, d->v_sh) ||
      (q && (!view_ok(d->q, d->q_sb, d->q_st, d->q_sh) || !view_ok(d->q_out, d->out_sb, d->out_st, d->out_sh)))) {
    set_error("%s: k, v, q and q_out must be 16-byte aligned with non-negative strides that are "
              "multiples of 8 elements", fn);
    return SKV_E_ARG;
  }
  if (!pool_ok(d->k_pool, d->v_pool)) {
    set_error("%s: pools must be 16-byte aligned", fn);
    return SKV_E_ARG;
  }
  if (d->half < 0 || d->half > kHeadDim / 2 || d->half % 8 || (d->half > 0) != (d->cos != nullptr) ||
      (d->cos == nullptr) != (d->sin == nullptr)) {
    set_error("%s: the rotation takes cos and sin of 8, 16 .. 64 columns, or neither", fn);
    return SKV_E_ARG;
  }
  if (d->half && (d->table_rows <= 0 || d->cos_stride < d->half || d->cos_stride % 4 ||
                  reinterpret_cast<uintptr_t>(d->cos) % 16 || reinterpret_cast<uintptr_t>(d->sin) % 16)) {
    set_error("%s: cos / sin need rows, 16-byte aligned pointers and a row stride that is a "
              "multiple of 4 and holds the columns", fn);
    return SKV_E_ARG;
  }
  const skv_head_norm* norms[2] = {&d->norm_q, &d->norm_k};
  for (const skv_head_norm* n : norms) {
    if (n->norm && (!(n->eps >= 0.0f) ||
                    (n->weight && (reinterpret_cast<uintptr_t>(n->weight) % 16 ||
                                   (n->weight_dtype != SKV_F32 && !half_dtype(n->weight_dtype)))))) {
      set_error("%s: norms need eps >= 0 and 16-byte aligned f32, bf16 or f16 weights", fn);
      return SKV_E_ARG;
    }
  }
  AppendPagesArgs a{};
  a.pg.tables = d->tables, a.pg.table_st = d->table_stride, a.pg.capacity = (int64_t)d->table_width * d->page_tokens;
  a.pg.n_pages = d->n_pages, a.pg.T = d->page_tokens, a.pg.Tp = padded_tokens(d->page_tokens);
  a.pg.heads = d->kv_heads, a.pg.lengths = d->lengths, a.pg.new_lens = d->new_lens;
  a.q = d->q, a.q_sb = d->q_sb, a.q_st = d->q_st, a.q_sh = d->q_sh;
  a.k = d->k, a.k_sb = d->k_sb, a.k_st = d->k_st, a.k_sh = d->k_sh;
  a.v = d->v, a.v_sb = d->v_sb, a.v_st = d->v_st, a.v_sh = d->v_sh;
  a.q_out = d->q_out, a.o_sb = d->out_sb, a.o_st = d->out_st, a.o_sh = d->out_sh;
  a.k_pool = d->k_pool, a.v_pool = d->v_pool;
  a.wq = d->norm_q.norm ? d->norm_q.weight : nullptr, a.wq_dtype = d->norm_q.weight_dtype;
  a.wk = d->norm_k.norm ? d->norm_k.weight : nullptr, a.wk_dtype = d->norm_k.weight_dtype;
  a.norm_q = d->norm_q.norm != 0, a.norm_k = d->norm_k.norm != 0;
  a.eps_q = d->norm_q.eps, a.eps_k = d->norm_k.eps;
  a.q_heads = d->q_heads, a.q_blocks = head_blocks(d->q_heads);
  a.k_blocks = head_blocks(d->kv_heads);
  a.cos = d->cos, a.sin = d->sin, a.tab_st = d->cos_stride, a.tab_rows = d->table_rows;
  a.pos = d->positions, a.pos_sb = d->pos_sb, a.pos_st = d->pos_st, a.pos0 = d->position0;
  a.pos64 = d->pos_is_int64, a.half = d->half, a.batch = d->batch, a.rows = d->rows;
  const int64_t tokens = (int64_t)d->batch * d->rows;
  if (tokens == 0) return SKV_OK;
  const int64_t units = tokens * (a.q_blocks + (int64_t)a.k_blocks), groups = (units + 15) / 16;
  if (groups * 256 >= kMaxThreads) {
    set_error("%s: too many rows (batch=%d rows=%d)", fn, d->batch, d->rows);
    return SKV_E_ARG;
  }
  const int64_t per_page = (d->page_tokens + kTile - 1) / kTile;
  const int64_t ends = ((int64_t)d->rows + d->page_tokens - 2) / d->page_tokens;  // page ends among the new tokens
  const int64_t by_tile = (d->rows - 1) / kTile + 2 + ends, by_page = (ends + 1) * per_page;
  a.v_tiles = (int)(by_tile < by_page ? by_tile : by_page);
  const int64_t v_groups = (int64_t)d->batch * d->kv_heads * a.v_tiles;
  if ((groups + v_groups) * 256 >= kMaxThreads) {
    set_error("%s: too many rows (batch=%d rows=%d)", fn, d->batch, d->rows);
    return SKV_E_ARG;
  }
  a.n_units_q = (int)(tokens * a.q_blocks);
  a.n_units = (int)units;
  a.n_unit_groups = (int)groups;
  const dim3 grid((unsigned)(groups + v_groups)), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->dtype == SKV_BF16) {
    if (d->interleaved) hipLaunchKernelGGL((append_pages_kernel<bf16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((append_pages_kernel<bf16, false>), grid, block, 0, s, a);
  } else {
    if (d->interleaved) hipLaunchKernelGGL((append_pages_kernel<f16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((append_pages_kernel<f16, false>), grid, block, 0, s, a);
  }
  return launched(fn);
}

extern "C" int skv_attend_shared_workspace(const skv_attend_shared_desc* d, int64_t* bytes) {
  const char* fn = "skv_attend_shared_workspace";
  int st = check_shared(fn, d);
  if (st != SKV_OK) return st;
  if (!bytes) {
    set_error("%s: null result", fn);
    return SKV_E_ARG;
  }
  SharedPlan p;
  st = plan_shared(fn, d, &p);
  if (st == SKV_OK) *bytes = p.bytes;
  return st;
}

extern "C" int skv_attend_shared(const skv_attend_shared_desc* d, skv_stream_t stream) {
  const char* fn = "skv_attend_shared";
  int st = check_shared(fn, d);
  if (st != SKV_OK) return st;
  SharedPlan p;
  st = plan_shared(fn, d, &p);
  if (st != SKV_OK) return st;
  if (d->batch == 0 || d->rows == 0) return SKV_OK;
  if (p.bytes > 0 && (!d->workspace || d->workspace_bytes < p.bytes ||
                      reinterpret_cast<uintptr_t>(d->workspace) % 16)) {
    set_error("%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)p.bytes);
    return SKV_E_ARG;
  }
  SharedArgs a{};
  a.q = d->q, a.q_sb = d->q_sb, a.q_st = d->q_st, a.q_sh = d->q_sh;
  a.out = d->out, a.o_sb = d->out_sb, a.o_st = d->out_st, a.o_sh = d->out_sh;
  a.own = Source{d->k_pool, d->v_pool, d->n_pages, d->page_tokens, padded_tokens(d->page_tokens)};
  if (d->prefix_tokens > 0)
    a.pre = Source{d->prefix_k_pool, d->prefix_v_pool, d->prefix_n_pages, d->prefix_page_tokens,
                   padded_tokens(d->prefix_page_tokens)};
  a.pre_pages = d->prefix_pages, a.pre_tokens = d->prefix_tokens;
  a.tables = d->tables, a.table_st = d->table_stride, a.width = d->table_width;
  a.lengths = d->lengths, a.new_lens = d->new_lens;
  a.batch = d->batch, a.rows = d->rows, a.heads = d->kv_heads, a.group = d->q_heads / d->kv_heads;
  a.causal = d->causal != 0, a.c = d->softmax_scale * 1.44269504088896340736f;
  a.M = d->batch * d->rows * a.group;
  a.pre_splits = p.pre_splits, a.pre_grid = p.pre_grid;
  a.own_rb = p.own_rb, a.own_splits = p.own_splits;
  a.own_items = p.own_items, a.own_waves = p.own_waves;
  a.direct = p.parts == 1, a.both = p.both;
  a.part_o = static_cast<float*>(d->workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (int64_t)p.parts * a.heads * a.M * kHeadDim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.parts > 0) {
    if (d->dtype == SKV_BF16) launch_shared<bf16>(a, p, s);
    else launch_shared<f16>(a, p, s);
    st = launched(fn);
    if (st != SKV_OK || a.direct) return st;
  }
  if (d->dtype == SKV_BF16) launch_merge<bf16>(a, p.parts, s);
  else launch_merge<f16>(a, p.parts, s);
  return launched(fn);
}
