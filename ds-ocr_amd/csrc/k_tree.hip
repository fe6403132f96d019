// k_tree.hip — drafted tokens over a KV cache: attention of a tree's nodes (k_tree_attend), verification of the drafts
// (k_tree_verify), and the accepted nodes' rows and weights into the cache (k_tree_commit).
#include "dsh.h"
#include "k_core.h"

#include <string.h>

#include <type_traits>

typedef unsigned long long u64;

// ---------------------------------------------------------------------------- the tree
// Every node's ancestors-or-self as 128 bits and its depth, from the parents, by pointer doubling: after round r a node
// knows its next 2^r ancestors, so that a chain of 128 takes 7 rounds. A padding node (a parent outside [-1, i), or a padding
// node above it) has no bits. Called by every thread of a block of at least DSH_TREE_MAX with its node's parent.
struct tree_lds {
  u64 anc[DSH_TREE_MAX][2];
  int up[DSH_TREE_MAX];
};
__device__ __forceinline__ int tree_parent(const int *parents, int n) {
  return (int)threadIdx.x < n ? parents[threadIdx.x] : -2;
}
__device__ void tree_ancestors(tree_lds &t, int up, int n) {
  const int i = threadIdx.x;
  u64 lo = 0, hi = 0;
  if (i < n) {
    if (up < -1 || up >= i) up = -2;
    lo = i < 64 ? 1ull << i : 0;
    hi = i < 64 ? 0 : 1ull << (i - 64);
    t.anc[i][0] = lo;
    t.anc[i][1] = hi;
    t.up[i] = up;
  }
  for (int span = 1; span < n; span *= 2) {
    __syncthreads();
    const bool more = i < n && up >= 0;
    if (more) {
      lo |= t.anc[up][0];
      hi |= t.anc[up][1];
      up = t.up[up];
    }
    __syncthreads();
    if (more) {
      t.anc[i][0] = lo;
      t.anc[i][1] = hi;
      t.up[i] = up;
    }
  }
  __syncthreads();
  if (i < n && up == -2) t.anc[i][0] = t.anc[i][1] = 0;
  __syncthreads();
}
__device__ __forceinline__ int tree_depth(const u64 *anc) { return __popcll(anc[0]) + __popcll(anc[1]) - 1; }

// ---------------------------------------------------------------------------- attention
// The rows of one key head are the (node, query head of its group) pairs, row r node r % n_nodes of head r / n_nodes. A wave
// owns 16 rows and goes over tiles of AT positions with a running maximum and sum, everything in registers:
//   S^T[position][row] = K Q^T: lane (i, g), i = lane & 15, g = lane >> 4, has row i of the K tile as the product's left
//   operand, and gets back row i of the queries at the positions 4g..4g+3 of a 16-position subtile;
//   O^T[dimension][row] += V^T P^T: that is just the right operand of the second product, whose summation index the lanes'
//   g and the four positions are. The order of the dimensions within a product and of its rows is free, so K and V are
//   loaded as they lie in memory: 16 bytes a lane, whole lines, no LDS and no exchange between lanes.
// The maximum is only moved, and the sums scaled, when some score exceeds it by ATT_SLACK: weights stay below exp(ATT_SLACK).
//   f32 cache: v_mfma_f32_16x16x4, exact products and f32 sums. bf16 cache: v_mfma_f32_16x16x32_bf16, the f32 queries and
//   weights in three bf16 parts each that add up to them exactly (24 bits), so that only the f32 sums round.
#define ATT_SLACK 10.0f
#define ATT_L2E 1.44269504088896340736f

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// How a launch cuts the work; a tile is AT positions of the cache (tiles in [gap, gap + skip) are seen by no node and left out)
// or of the tree.
struct attend_plan {
  int tile_rows, pos_waves;  // 16-row tiles and shares of the positions in a block: a wave each
  int groups, splits;        // blocks per key head: groups of tile_rows tiles of rows, splits of the tiles of positions
  int staged;                // k_tree_attend_rows
  int cache_tiles, tree_tiles, gap, skip, per;  // per: tiles of a split
  int grp;                                       // query heads per key head
  float inv_nodes;                               // 1 / n_nodes
  float *part, *ml;          // [head][group][split][16 * tile_rows] x D, and the maximum and sum
};

__device__ __forceinline__ float att_exp(float x) { return __builtin_amdgcn_exp2f(x * ATT_L2E); }

// x as three bf16 numbers whose sum it is (each the upper half of what is left: 8 + 8 + 8 bits), in the upper halves.
__device__ __forceinline__ void split3(float x, uint32_t &a, uint32_t &b, uint32_t &c) {
  a = __float_as_uint(x) & 0xFFFF0000u;
  const float r = x - __uint_as_float(a);
  b = __float_as_uint(r) & 0xFFFF0000u;
  c = __float_as_uint(r - __uint_as_float(b));
}
// The upper halves of lo and hi, side by side.
__device__ __forceinline__ uint32_t upper2(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

template <int D>
struct frag_f32 {
  static constexpr int AT = 16, NB = D / 16;
  f32x4 q[NB], k[NB], v[4][D / 64];
  __device__ __forceinline__ void load_q(const float *p, int g) {
#pragma unroll
    for (int b = 0; b < NB; b++) q[b] = *(const f32x4 *)(p + 16 * b + 4 * g);
  }
  // row(x): element offset of the tile's position x
  template <typename R>
  __device__ __forceinline__ void load_k(const void *base, R row, int i, int g) {
    const float *p = (const float *)base + row(i) + 4 * g;
#pragma unroll
    for (int b = 0; b < NB; b++) k[b] = *(const f32x4 *)(p + 16 * b);
  }
  template <typename R>
  __device__ __forceinline__ void load_v(const void *base, R row, int i, int g) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const float *p = (const float *)base + row(4 * g + r) + 4 * i;
#pragma unroll
      for (int b = 0; b < D / 64; b++) v[r][b] = *(const f32x4 *)(p + 64 * b);
    }
  }
  __device__ __forceinline__ void scores(float *s) const {
    f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f}, c = a;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[b][e], q[b][e], a, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(k[b][e + 1], q[b][e + 1], c, 0, 0, 0);
      }
#pragma unroll
    for (int r = 0; r < 4; r++) s[r] = a[r] + c[r];
  }
  __device__ __forceinline__ void add(const float *p, f32x4 *o) const {
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int b = 0; b < D / 64; b++)
#pragma unroll
        for (int t = 0; t < 4; t++) o[4 * b + t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][b][t], p[r], o[4 * b + t], 0, 0, 0);
  }
  // Whether position x of the lane's (4g + x) holds a value that is not finite here; and takes it out.
  __device__ __forceinline__ bool clean_v(int x) {
    bool bad = false;
#pragma unroll
    for (int b = 0; b < D / 64; b++)
#pragma unroll
      for (int t = 0; t < 4; t++)
        if (!(__builtin_fabsf(v[x][b][t]) < __builtin_huge_valf())) {
          bad = true;
          v[x][b][t] = 0.0f;
        }
    return bad;
  }
  // Dimension of o[4b + t][r].
  static __device__ __forceinline__ int dim(int b, int r, int g) { return 64 * b + 16 * g + 4 * r; }
};

// Output in registers: o[4b + t][r] is dimension dim(b, r, g) + t of the lane's row.
template <int D>
struct frag_bf16 {
  static constexpr int AT = 32, NS = D / 32;
  u32x4 q[3][NS], k[2][NS];
  uint32_t v[8][D / 32];  // position 16 (x >> 2) + 4g + (x & 3), D / 64 groups of four dimensions
  __device__ __forceinline__ void load_q(const float *p, int g) {
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const f32x4 x0 = *(const f32x4 *)(p + 32 * s + 8 * g), x1 = *(const f32x4 *)(p + 32 * s + 8 * g + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        uint32_t a[2], b[2], c[2];
        split3(e < 2 ? x0[2 * e] : x1[2 * e - 4], a[0], b[0], c[0]);
        split3(e < 2 ? x0[2 * e + 1] : x1[2 * e - 3], a[1], b[1], c[1]);
        q[0][s][e] = upper2(a[0], a[1]);
        q[1][s][e] = upper2(b[0], b[1]);
        q[2][s][e] = upper2(c[0], c[1]);
      }
    }
  }
  template <typename R>
  __device__ __forceinline__ void load_k(const void *base, R row, int i, int g) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint16_t *p = (const uint16_t *)base + row(16 * h + i) + 8 * g;
#pragma unroll
      for (int s = 0; s < NS; s++) k[h][s] = *(const u32x4 *)(p + 32 * s);
    }
  }
  template <typename R>
  __device__ __forceinline__ void load_v(const void *base, R row, int i, int g) {
#pragma unroll
    for (int x = 0; x < 8; x++) {
      const uint16_t *p = (const uint16_t *)base + row(16 * (x >> 2) + 4 * g + (x & 3)) + 4 * i;
#pragma unroll
      for (int b = 0; b < D / 64; b++) {
        const uint2 w = *(const uint2 *)(p + 64 * b);
        v[x][2 * b] = w.x;
        v[x][2 * b + 1] = w.y;
      }
    }
  }
  __device__ __forceinline__ void scores(float *s) const {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int l = 2; l >= 0; l--)  // the small parts first
#pragma unroll
        for (int x = 0; x < NS; x++)
          a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[h][x]), __builtin_bit_cast(bf16x8, q[l][x]),
                                                      a, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; r++) s[4 * h + r] = a[r];
    }
  }
  __device__ __forceinline__ void add(const float *p, f32x4 *o) const {
    u32x4 w[3];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      uint32_t a[2], b[2], c[2];
      split3(p[2 * e], a[0], b[0], c[0]);
      split3(p[2 * e + 1], a[1], b[1], c[1]);
      w[0][e] = upper2(a[0], a[1]);
      w[1][e] = upper2(b[0], b[1]);
      w[2][e] = upper2(c[0], c[1]);
    }
#pragma unroll
    for (int b = 0; b < D / 64; b++)
#pragma unroll
      for (int t = 0; t < 4; t++) {
        u32x4 x;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t lo = v[2 * e][2 * b + (t >> 1)], hi = v[2 * e + 1][2 * b + (t >> 1)];
          x[e] = __builtin_amdgcn_perm(hi, lo, t & 1 ? 0x07060302u : 0x05040100u);
        }
#pragma unroll
        for (int l = 2; l >= 0; l--)
          o[4 * b + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w[l]),
                                                                 o[4 * b + t], 0, 0, 0);
      }
  }
  __device__ __forceinline__ bool clean_v(int x) {
    bool bad = false;
#pragma unroll
    for (int b = 0; b < D / 32; b++) {
      if ((v[x][b] & 0x7F80u) == 0x7F80u) bad = true, v[x][b] &= 0xFFFF0000u;
      if ((v[x][b] & 0x7F800000u) == 0x7F800000u) bad = true, v[x][b] &= 0xFFFFu;
    }
    return bad;
  }
  static __device__ __forceinline__ int dim(int b, int r, int g) { return 64 * b + 16 * g + 4 * r; }
};

// A block: tile_rows x pos_waves waves over one split of the tiles of one key head; the waves of a row tile put their sums
// together, and the block writes them for k_tree_join (splits > 1) or finishes its rows itself. Up to a few hundred rows the
// launches and the first loads' round trips are all (5 nodes over 77 rows 8.4 us, 16 over 701 11.5 with the join's 3); then
// the cache's bytes (10 heads x 128: 7001 rows 18.6 us for one node, 20 for 16, 72 MB; 30000 rows 61 us, 307 MB, 5.0 TB/s).
template <int D, bool BF>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) k_tree_attend(dsh_tree_attn_t A, attend_plan P) {
  typedef typename std::conditional<BF, frag_bf16<D>, frag_f32<D>>::type frag;
  constexpr int AT = frag::AT, NV = AT / 4;  // scores a lane
  __shared__ tree_lds t;
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ bool s_live[32];
  extern __shared__ __attribute__((aligned(16))) float s_o[];  // pos_waves > 1: [wave][16][min(D, 128) + 4]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const int T = A.n_nodes, R = T * P.grp;
  const int kh = blockIdx.y, z = blockIdx.z, split = blockIdx.x;
  const int pw = P.pos_waves == 4 ? wave : P.pos_waves == 2 ? wave >> 1 : 0, rt = wave - pw * P.tile_rows;
  const int row = 16 * (z * P.tile_rows + rt) + i;  // the lane's
  const int rr = min(row, R - 1), rh = (int)(((float)rr + 0.5f) * P.inv_nodes);  // 2^17 rows at most: exact
  const int node = rr - rh * T, head = kh * P.grp + rh;
  const int tiles = P.cache_tiles - P.skip + P.tree_tiles, t0 = split * P.per, t1 = min(t0 + P.per, tiles);
  // what only the tree's own tiles, a window, scores and whole rows need
  const bool need = P.splits == 1 || A.scores || A.window > 0 || t1 > P.cache_tiles - P.skip;
  const int parent = need ? tree_parent(A.parents, T) : -2;
  frag F;
  // a tile: its rows (the cache's or the tree's own) and how many there are; loads past them repeat the last one
  struct where {
    const void *k, *v;
    int64_t rs;
    int p0, end;
    bool own;
    __device__ __forceinline__ int64_t operator()(int x) const { return min(p0 + x, end - 1) * rs; }
  };
  const auto locate = [&](int tile) {
    const int x = tile >= P.gap ? tile + P.skip : tile;
    const bool own = x >= P.cache_tiles;
    const dsh_kv_t &c = own ? A.tree : A.cache;
    const int64_t h = kh * c.head_stride * (BF ? 2 : 4);
    return where{(const char *)c.k + h, (const char *)c.v + h, c.row_stride, AT * (own ? x - P.cache_tiles : x),
                 own ? T : A.n_cache, own};
  };
  where nx = locate(min(t0 + pw, tiles - 1));
  F.load_q(A.q + node * A.q_stride + (int64_t)head * D, g);
  F.load_k(nx.k, nx, i, g);
  F.load_v(nx.v, nx, i, g);
  if (need) tree_ancestors(t, parent, T);
  const u64 anc0 = need ? t.anc[node][0] : 0, anc1 = need ? t.anc[node][1] : 0;
  const bool live = !need || (anc0 | anc1);
  // the lane's row sees the positions below prefill_len and from lo on (all of them without a window)
  const int pos = A.n_cache + __popcll(anc0) + __popcll(anc1) - 1;
  const int lo = A.window > 0 && pos >= A.prefill_len ? max(A.prefill_len, pos + 1 - A.window) : 0;
  const float inf = __builtin_huge_valf();
  float m = -inf, l = 0.0f, ml2 = 0.0f;
  f32x4 o[D / 16];
#pragma unroll
  for (int b = 0; b < D / 16; b++) o[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float *sc = A.scores ? A.scores + ((int64_t)head * T + node) * A.score_stride : nullptr;

  const int lo_most = A.n_cache + T - A.window;  // from here on every node's window holds a row
  for (int tile = t0 + pw; tile < t1; tile += P.pos_waves) {
    const bool own = nx.own;
    const int p0 = nx.p0, end = nx.end;
    float s[NV];
    F.scores(s);
    // the next tile's K while this one's V is on its way, then its V; without a branch (past the end the last tile
    // again), so that the waits are counted and neither waits for the other
    nx = locate(min(tile + P.pos_waves, tiles - 1));
    F.load_k(nx.k, nx, i, g);
#pragma unroll
    for (int k = 0; k < NV; k++) s[k] *= A.scale;
    if (own || p0 + AT > end || (A.window > 0 && p0 + AT > A.prefill_len && p0 < lo_most)) {
      // some position is not seen by some row
      uint32_t seen = 0;
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int j = p0 + 16 * (k >> 2) + 4 * g + (k & 3);
        bool see = live && j < end;
        int p = j;
        if (own) {
          const int a = min(j, DSH_TREE_MAX - 1);
          see = see && (((a < 64 ? anc0 >> a : anc1 >> (a - 64)) & 1) != 0);
          if (A.window > 0) p = A.n_cache + tree_depth(t.anc[a]);
        }
        see = see && (p < A.prefill_len || p >= lo);
        s[k] = see ? s[k] : -inf;
        seen |= (uint32_t)see << k;
      }
      // A weight of 0 does not take out a V that is not finite: such rows are set to 0, and what sees them to NaN. (At the
      // cache's end what stands in for the rows behind it is its last row, which every node sees.)
      if (own || A.window > 0) {
        bool poison = false;
#pragma unroll
        for (int k = 0; k < NV; k++) {
          const u64 bad = __ballot(F.clean_v(k));
          poison |= ((bad >> (16 * g)) & 0xFFFF) && ((seen >> k) & 1);
        }
        if (__any(poison)) {
          int y = poison;
          y |= __shfl_xor(y, 16);
          y |= __shfl_xor(y, 32);
          if (y)
#pragma unroll
            for (int b = 0; b < D / 16; b++) o[b] += __builtin_nanf("");
        }
      }
    }
    if (sc && row < R) {
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int j = p0 + 16 * (k >> 2) + 4 * g + (k & 3);
        if (j < end) sc[own ? (int64_t)A.n_cache + j : j] = live ? s[k] : -inf;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int k = 1; k < NV; k++) mx = fmaxf(mx, s[k]);
    if (__any(mx > m + ATT_SLACK)) {
      mx = fmaxf(mx, m);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float f = mx == m ? 1.0f : att_exp(m - mx);
      m = mx;
      ml2 = m == -inf ? 0.0f : m * ATT_L2E;
      l *= f;
#pragma unroll
      for (int b = 0; b < D / 16; b++) o[b] *= f;
    }
#pragma unroll
    for (int k = 0; k < NV; k++) {
      s[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], ATT_L2E, -ml2));
      l += s[k];
    }
    F.add(s, o);
    F.load_v(nx.v, nx, i, g);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // A row's sums, for the join or finished: factor * (what the waves of its tile have).
  const auto put = [&](int node, int head, int64_t at, int d, f32x4 y, float m, float l, bool live) {
    if (P.splits > 1) {
      *(f32x4 *)(P.part + at * D + d) = y;
      if (d == 0) *(f32x2 *)(P.ml + 2 * at) = f32x2{m, l};
      return;
    }
    const bool none = !live || l == 0.0f;
    y = none ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : y * (1.0f / l);
    *(f32x4 *)(A.out + node * A.out_stride + (int64_t)head * D + d) = y;
    if (A.lse && d == 0) A.lse[(int64_t)head * T + node] = none ? -inf : m + logf(l);
  };
  const int64_t at0 = (((int64_t)kh * P.groups + z) * P.splits + split) * 16 * P.tile_rows;
  if (P.pos_waves == 1) {
    if (row >= R) return;
#pragma unroll
    for (int b = 0; b < D / 64; b++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        put(node, head, at0 + 16 * rt + i, frag::dim(b, r, g), f32x4{o[4 * b][r], o[4 * b + 1][r], o[4 * b + 2][r], o[4 * b + 3][r]},
            m, l, live);
    return;
  }
  // the waves of a row tile: every thread of the block adds up pieces of four dimensions
  if (g == 0) {
    s_m[wave][i] = m;
    s_l[wave][i] = l;
    s_live[16 * rt + i] = live;
  }
  constexpr int CH = D < 128 ? D : 128;  // dimensions at a time, for the LDS
#pragma unroll
  for (int c = 0; c < D; c += CH) {
    const int width = min(CH, D - c);
    if (c) __syncthreads();
#pragma unroll
    for (int b = c / 64; b < (c + CH) / 64 && b < D / 64; b++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        *(f32x4 *)(s_o + (wave * 16 + i) * (CH + 4) + frag::dim(b, r, g) - c) =
            f32x4{o[4 * b][r], o[4 * b + 1][r], o[4 * b + 2][r], o[4 * b + 3][r]};
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * P.tile_rows * (width / 4); x += 256) {
      const int r = x / (width / 4), d = 4 * (x - r * (width / 4)), r16 = r & 15, tile = r >> 4, row = 16 * z * P.tile_rows + r;
      if (row >= R) continue;
      float M = -inf, L = 0.0f;
      for (int w = 0; w < P.pos_waves; w++) M = fmaxf(M, s_m[w * P.tile_rows + tile][r16]);
      f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int w = 0; w < P.pos_waves; w++) {
        const int v = w * P.tile_rows + tile;
        const float mw = s_m[v][r16], f = mw == M ? 1.0f : att_exp(mw - M);
        L += s_l[v][r16] * f;
        y += *(const f32x4 *)(s_o + (v * 16 + r16) * (CH + 4) + d) * f;
      }
      const int h = (int)(((float)row + 0.5f) * P.inv_nodes), nd = row - h * T;
      put(nd, kh * P.grp + h, at0 + r, c + d, y, M, L, s_live[r]);
    }
  }
}

// The same where a key head has many rows: a block of eight waves, up to eight 16-row tiles, shares tiles of 32 positions through
// LDS. With an f32 cache the products are bf16 ones as well, of three parts a number (split3) and without the three smallest
// of the nine pairs (2^-21 of the product at most, all that is left out): 6 x 16 cycles where v_mfma_f32_16x16x4 takes 8 x 32,
// and the parts are made once a block, when what was loaded is written to LDS. K lies there as rows of 16-byte pieces, V
// transposed, 32 positions of a dimension in 64 bytes in the order of the summation index; both with the pieces' places
// exclusive-ored so that the 16 lanes of a read or write meet all banks. The last SW waves bring the next tile into the other
// half of the LDS while the others compute, one of each kind to a SIMD, so that the vector units' splitting and the matrix
// units' products go on at once; where there are rows for all eight (SW = 8), each does both, half of them in the other order.
// What bounds it is the length of a tile's steps in a wave (LDS reads, products, weights, products): 64 nodes over 7001 rows 23 us
// and 5 for the join, against 37 and 5 in k_tree_attend with f32 products; 24 nodes of 16 heads over 120011 bf16 rows 84 us
// (246 MB, 2.9 TB/s; 820 TFLOP/s of bf16 products) and 5, against 147. Two row tiles to a wave (half the LDS reads) spill and
// take 43 and 150 us, 64 positions a step 126 with the bf16 cache.
template <int D, bool BF>
struct staged {
  static constexpr int NL = BF ? 1 : 3, E = BF ? 8 : 4;  // parts; dimensions of a unit: 4 positions x E, 16 bytes a position
  static constexpr int UNITS = 8 * (D / E);              // of K, and again of V
  uint8_t k[NL][32 * D * 2], v[NL][D * 64];
  static __device__ __forceinline__ int k_at(int row, int piece) {
    const int x = D % 128 == 0 ? row & 15 : (row >> 1) & 7;
    return row * 2 * D + 16 * (piece ^ x);
  }
  static __device__ __forceinline__ int v_at(int d, int g) {
    const int c = d >> 2;
    return c * 256 + 16 * (((d & 3) * 4 + g) ^ ((c ^ (c >> 4)) & 15));
  }
};

template <int D, bool BF, int SW>
__global__ void __launch_bounds__(512) k_tree_attend_rows(dsh_tree_attn_t A, attend_plan P) {
  typedef staged<D, BF> stage;
  constexpr int NL = stage::NL, E = stage::E, UNITS = stage::UNITS, SN = 64 * SW, U = (2 * UNITS + SN - 1) / SN, NS = D / 32;
  constexpr int AHEAD = U * (BF ? 3 : 2) <= 8 ? BF ? 3 : 2 : 1;  // tiles on their way, in registers
  __shared__ __attribute__((aligned(1024))) stage S[2];
  __shared__ uint32_t s_bad[3];  // by the tile: positions with a V that is not finite (where some row does not see all of it)
  __shared__ tree_lds t;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
  const int T = A.n_nodes, R = T * P.grp, kh = blockIdx.y, z = blockIdx.z, split = blockIdx.x, rt = wave;
  const bool works = rt < P.tile_rows, stager = wave >= 8 - SW;
  const int sid = tid - 64 * (8 - SW);
  const int row = 16 * (z * P.tile_rows + rt) + i;
  const int rr = min(row, R - 1), rh = (int)(((float)rr + 0.5f) * P.inv_nodes), node = rr - rh * T, head = kh * P.grp + rh;
  const int tiles = P.cache_tiles - P.skip + P.tree_tiles, t0 = split * P.per, t1 = min(t0 + P.per, tiles);
  const bool need = P.splits == 1 || A.scores || A.window > 0 || t1 > P.cache_tiles - P.skip;
  const int parent = need ? tree_parent(A.parents, T) : -2;
  struct where {
    const char *k, *v;
    int64_t rs;
    int p0, end;
    bool own;
  };
  const auto locate = [&](int tile) {
    const int x = tile >= P.gap ? tile + P.skip : tile;
    const bool own = x >= P.cache_tiles;
    const dsh_kv_t &c = own ? A.tree : A.cache;
    const int64_t h = kh * c.head_stride * (BF ? 2 : 4);
    return where{(const char *)c.k + h, (const char *)c.v + h, c.row_stride * (BF ? 2 : 4), 32 * (own ? x - P.cache_tiles : x),
                 own ? T : A.n_cache, own};
  };
  // the thread's units of a tile: unit u = sid + SN y, K's before V's; quad q of the positions, dimensions E c...
  const auto load = [&](u32x4 (*st)[4], const where &w) {
    const int64_t r1 = w.rs, r3 = 3 * w.rs;
    const bool whole = w.p0 + 32 <= w.end;
#pragma unroll
    for (int y = 0; y < U; y++) {
      const int u = sid + SN * y;
      if (2 * UNITS % SN && u >= 2 * UNITS) continue;
      const bool is_v = UNITS % SN ? u >= UNITS : y >= UNITS / SN;
      const int x = is_v ? u - UNITS : u, q = x / (D / E), c = x - q * (D / E);
      const char *b = (is_v ? w.v : w.k) + 16 * c;
      if (whole) {
        const char *p = b + w.p0 * w.rs + 4 * q * w.rs;
        st[y][0] = *(const u32x4 *)p;
        st[y][1] = *(const u32x4 *)(p + r1);
        st[y][2] = *(const u32x4 *)(p + 2 * r1);
        st[y][3] = *(const u32x4 *)(p + r3);
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++) st[y][r] = *(const u32x4 *)(b + min(w.p0 + 4 * q + r, w.end - 1) * w.rs);
      }
    }
  };
  const auto write = [&](u32x4 (*st)[4], stage &S, bool part, uint32_t *bad_word) {
#pragma unroll
    for (int y = 0; y < U; y++) {
      const int u = sid + SN * y;
      if (2 * UNITS % SN && u >= 2 * UNITS) continue;
      const bool is_v = UNITS % SN ? u >= UNITS : y >= UNITS / SN;
      const int x = is_v ? u - UNITS : u, q = x / (D / E), c = x - q * (D / E);
      if (part && is_v) {  // what is not finite becomes 0: see k_tree_attend
#pragma unroll
        for (int r = 0; r < 4; r++) {
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (BF) {
              if ((st[y][r][e] & 0x7F80u) == 0x7F80u) bad = true, st[y][r][e] &= 0xFFFF0000u;
              if ((st[y][r][e] & 0x7F800000u) == 0x7F800000u) bad = true, st[y][r][e] &= 0xFFFFu;
            } else if ((st[y][r][e] & 0x7F800000u) == 0x7F800000u) {
              bad = true;
              st[y][r][e] = 0;
            }
          }
          if (bad) atomicOr(bad_word, 1u << (4 * q + r));
        }
      }
      if (BF) {
        if (!is_v) {
#pragma unroll
          for (int r = 0; r < 4; r++) *(u32x4 *)(S.k[0] + stage::k_at(4 * q + r, c)) = st[y][r];
        } else {
#pragma unroll
          for (int d = 0; d < 8; d++) {
            const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
            uint2 w;
            w.x = __builtin_amdgcn_perm(st[y][1][d >> 1], st[y][0][d >> 1], sel);
            w.y = __builtin_amdgcn_perm(st[y][3][d >> 1], st[y][2][d >> 1], sel);
            *(uint2 *)(S.v[0] + stage::v_at(8 * c + d, q & 3) + 8 * (q >> 2)) = w;
          }
        }
      } else {
        uint32_t a[3][4][4];  // part, position, dimension
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int e = 0; e < 4; e++) split3(__uint_as_float(st[y][r][e]), a[0][r][e], a[1][r][e], a[2][r][e]);
#pragma unroll
        for (int n = 0; n < NL; n++) {
          if (!is_v) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
              uint2 w;
              w.x = upper2(a[n][r][0], a[n][r][1]);
              w.y = upper2(a[n][r][2], a[n][r][3]);
              *(uint2 *)(S.k[n] + stage::k_at(4 * q + r, c >> 1) + 8 * (c & 1)) = w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              uint2 w;
              w.x = upper2(a[n][0][e], a[n][1][e]);
              w.y = upper2(a[n][2][e], a[n][3][e]);
              *(uint2 *)(S.v[n] + stage::v_at(4 * c + e, q & 3) + 8 * (q >> 2)) = w;
            }
          }
        }
      }
    }
  };
  const int lo_most = A.n_cache + T - A.window;
  // whether some row may not see all of a tile
  const auto partial = [&](const where &w) {
    return w.own || w.p0 + 32 > w.end || (A.window > 0 && w.p0 + 32 > A.prefill_len && w.p0 < lo_most);
  };
  u32x4 ahead[AHEAD][U][4];
  if (stager) {
#pragma unroll
    for (int a = 0; a < AHEAD; a++) load(ahead[a], locate(min(t0 + a, tiles - 1)));
  }
  // Tile t0 + n (n % AHEAD == a) to its half of the LDS, and the loads of the tile AHEAD after it.
  const auto bring = [&](int n, u32x4 (*st)[4]) {
    const where w = locate(t0 + n);
    write(st, S[n & 1], partial(w) && (w.own || A.window > 0), &s_bad[n % 3]);
    if (sid == 0) s_bad[(n + 1) % 3] = 0;  // read two tiles ago
    load(st, locate(min(t0 + n + AHEAD, tiles - 1)));
  };
  if (tid < 3) s_bad[tid] = 0;
  if (need) tree_ancestors(t, parent, T);
  const int count = t1 - t0;
  if (SW < 8 && stager) {
    __syncthreads();
    bring(0, ahead[0]);
    __syncthreads();
    // Whole rounds, with no way past a load: a tile's write then waits for its own loads, not for those behind them too (64
    // nodes over 7001 f32 rows 25.5 us with the join, 27.7 with the loads behind a condition).
    int n = 1;
    for (; n + AHEAD <= count; n += AHEAD)
#pragma unroll
      for (int a = 0; a < AHEAD; a++) {
        bring(n + a, ahead[(a + 1) % AHEAD]);
        __syncthreads();
      }
#pragma unroll
    for (int a = 0; a < AHEAD; a++)
      if (n + a < count) {
        bring(n + a, ahead[(a + 1) % AHEAD]);
        __syncthreads();
      }
    __syncthreads();
    return;
  }
  // the wave's queries, in three parts
  u32x4 qf[3][NS];
  {
    const float *p = A.q + node * A.q_stride + (int64_t)head * D + 8 * g;
#pragma unroll
    for (int x = 0; x < NS; x++) {
      float y[8];
      *(f32x4 *)y = *(const f32x4 *)(p + 32 * x);
      *(f32x4 *)(y + 4) = *(const f32x4 *)(p + 32 * x + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        uint32_t a[3], b[3];
        split3(y[2 * e], a[0], a[1], a[2]);
        split3(y[2 * e + 1], b[0], b[1], b[2]);
#pragma unroll
        for (int n = 0; n < 3; n++) qf[n][x][e] = upper2(a[n], b[n]);
      }
    }
  }
  const u64 anc0 = need ? t.anc[node][0] : 0, anc1 = need ? t.anc[node][1] : 0;
  const bool live = !need || (anc0 | anc1);
  const int pos = A.n_cache + __popcll(anc0) + __popcll(anc1) - 1;
  const int lo = A.window > 0 && pos >= A.prefill_len ? max(A.prefill_len, pos + 1 - A.window) : 0;
  const float inf = __builtin_huge_valf();
  float m = -inf, l = 0.0f, ml2 = 0.0f;
  f32x4 o[D / 16];  // o[b][r]: dimension 16 b + 4 g + r of the lane's row
#pragma unroll
  for (int b = 0; b < D / 16; b++) o[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float *sc = A.scores ? A.scores + ((int64_t)head * T + node) * A.score_stride : nullptr;
#define MFMA(a, b, c) \
  __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0)
  const auto compute = [&](int tile) {
    const where now = locate(t0 + tile);
    const bool own = now.own, part = partial(now);
    const int p0 = now.p0, end = now.end;
    float s[8];
    constexpr bool EARLY = BF && D <= 128;  // all of a tile's reads from LDS ahead of their use, where registers allow
    u32x4 f[2][EARLY ? NS : 1][NL], fv[EARLY ? D / 16 : 1][NL];
    // Places in LDS: of a row's and a dimension's first piece; the others' differ in bits, not in a sum, so an exclusive or and
    // an immediate give them. Opaque in every tile, or each is a register for the whole loop and some of them are
    // spilled (24 nodes of 16 heads over 120011 bf16 rows 86 us with the join, then 90; 32 over 40000 of 256 dimensions 113 and 232).
    constexpr int BITS = D % 128 ? 1 : 3;
    uint32_t k_0 = (tile & 1) * (uint32_t)sizeof(stage) + stage::k_at(i, g);
    uint32_t v_0 = (tile & 1) * (uint32_t)sizeof(stage) + (uint32_t)sizeof(S[0].k) + stage::v_at(i, g);
    __asm__("" : "+v"(k_0), "+v"(v_0));
    const auto read_k = [&](int h, int x) {
      const uint8_t *p = (const uint8_t *)S + (k_0 ^ (64 * (x & BITS))) + 64 * (x & ~BITS) + 32 * D * h;
#pragma unroll
      for (int n = 0; n < NL; n++) f[h][EARLY ? x : 0][n] = *(const u32x4 *)(p + n * sizeof S[0].k[0]);
    };
    const auto read_v = [&](int b) {
      const uint8_t *p = (const uint8_t *)S + (v_0 ^ (64 * (b & 3) + 16 * (b >> 2))) + 1024 * b;
#pragma unroll
      for (int n = 0; n < NL; n++) fv[EARLY ? b : 0][n] = *(const u32x4 *)(p + n * sizeof S[0].v[0]);
    };
    if (EARLY) {
#pragma unroll
      for (int x = 0; x < NS; x++) read_k(0, x), read_k(1, x);
#pragma unroll
      for (int b = 0; b < D / 16; b++) read_v(b);
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x4 a[2][2];
#pragma unroll
    for (int h = 0; h < 2; h++) a[h][0] = a[h][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < NS; x++) {
      if (!EARLY) read_k(0, x), read_k(1, x);
#pragma unroll
      for (int sum = 2; sum >= 0; sum--)  // the small products first
#pragma unroll
        for (int n = 0; n < NL; n++)
          if (sum - n >= 0 && sum - n < 3)
#pragma unroll
            for (int h = 0; h < 2; h++) a[h][x & 1] = MFMA(f[h][EARLY ? x : 0][n], qf[sum - n][x], a[h][x & 1]);
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) s[4 * h + r] = (a[h][0][r] + a[h][1][r]) * A.scale;
    if (part) {
      const uint32_t bad = s_bad[tile % 3];
      bool poison = false;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int at = 16 * (k >> 2) + 4 * g + (k & 3), j = p0 + at;
        bool see = live && j < end;
        int p = j;
        if (own) {
          const int a = min(j, DSH_TREE_MAX - 1);
          see = see && (((a < 64 ? anc0 >> a : anc1 >> (a - 64)) & 1) != 0);
          if (A.window > 0) p = A.n_cache + tree_depth(t.anc[a]);
        }
        see = see && (p < A.prefill_len || p >= lo);
        s[k] = see ? s[k] : -inf;
        poison |= see && ((bad >> at) & 1);
      }
      if (__any(poison)) {
        int y = poison;
        y |= __shfl_xor(y, 16);
        y |= __shfl_xor(y, 32);
        if (y)
#pragma unroll
          for (int b = 0; b < D / 16; b++) o[b] += __builtin_nanf("");
      }
    }
    if (sc && row < R) {
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int j = p0 + 16 * (k >> 2) + 4 * g + (k & 3);
        if (j < end) sc[own ? (int64_t)A.n_cache + j : j] = live ? s[k] : -inf;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int k = 1; k < 8; k++) mx = fmaxf(mx, s[k]);
    if (__any(mx > m + ATT_SLACK)) {
      mx = fmaxf(mx, m);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float f = mx == m ? 1.0f : att_exp(m - mx);
      m = mx;
      ml2 = m == -inf ? 0.0f : m * ATT_L2E;
      l *= f;
#pragma unroll
      for (int b = 0; b < D / 16; b++) o[b] *= f;
    }
    u32x4 pf[3];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      uint32_t a[3], b[3];
#pragma unroll
      for (int k = 2 * e; k < 2 * e + 2; k++) {
        s[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], ATT_L2E, -ml2));
        l += s[k];
      }
      split3(s[2 * e], a[0], a[1], a[2]);
      split3(s[2 * e + 1], b[0], b[1], b[2]);
#pragma unroll
      for (int n = 0; n < 3; n++) pf[n][e] = upper2(a[n], b[n]);
    }
#pragma unroll
    for (int b = 0; b < D / 16; b++) {
      if (!EARLY) read_v(b);
#pragma unroll
      for (int sum = 2; sum >= 0; sum--)
#pragma unroll
        for (int n = 0; n < NL; n++)
          if (sum - n >= 0 && sum - n < 3) o[b] = MFMA(fv[EARLY ? b : 0][n], pf[sum - n], o[b]);
    }
  };
  // one barrier a tile: tile n is read while tile n + 1 is written to the other half
  __syncthreads();
  if (SW == 8) {
    bring(0, ahead[0]);
    __syncthreads();
    for (int n0 = 0; n0 < count; n0 += AHEAD)
#pragma unroll
      for (int a = 0; a < AHEAD; a++) {
        const int n = n0 + a;
        if (n >= count) break;
        if (n + 1 < count && wave >= 4) bring(n + 1, ahead[(a + 1) % AHEAD]);
        if (works) compute(n);
        if (n + 1 < count && wave < 4) bring(n + 1, ahead[(a + 1) % AHEAD]);
        __syncthreads();
      }
  } else {
    __syncthreads();
    for (int n = 0; n < count; n++) {
      if (works) compute(n);
      __syncthreads();
    }
  }
#undef MFMA
  if (!works || row >= R) return;
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (P.splits > 1) {
    const int64_t at = (((int64_t)kh * P.groups + z) * P.splits + split) * 16 * P.tile_rows + 16 * rt + i;
#pragma unroll
    for (int b = 0; b < D / 16; b++) *(f32x4 *)(P.part + at * D + 16 * b + 4 * g) = o[b];
    if (g == 0) *(f32x2 *)(P.ml + 2 * at) = f32x2{m, l};
    return;
  }
  const bool none = !live || l == 0.0f;
#pragma unroll
  for (int b = 0; b < D / 16; b++)
    *(f32x4 *)(A.out + node * A.out_stride + (int64_t)head * D + 16 * b + 4 * g) =
        none ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o[b] * (1.0f / l);
  if (A.lse && g == 0) A.lse[(int64_t)head * T + node] = none ? -inf : m + logf(l);
}

// The splits of one row put together: a block per row, D / 4 threads to a split, 1024 / D splits at a time in their order.
template <int D>
__global__ void __launch_bounds__(256) k_tree_join(dsh_tree_attn_t A, attend_plan P) {
  constexpr int L = D / 4, N = 256 / L;
  __shared__ tree_lds t;
  __shared__ float s_f[1024], s_inv;
  __shared__ __attribute__((aligned(16))) float s_o[N][D];
  const int T = A.n_nodes, row = blockIdx.x, kh = blockIdx.y, rh = (int)(((float)row + 0.5f) * P.inv_nodes);
  const int node = row - rh * T, head = kh * P.grp + rh;
  const int z = (row >> 4) / P.tile_rows, in = row - z * 16 * P.tile_rows, stride = 16 * P.tile_rows;
  const int64_t at = ((int64_t)kh * P.groups + z) * P.splits * stride + in;
  const int parent = tree_parent(A.parents, T);
  const int x = threadIdx.x / L, d = 4 * (threadIdx.x - x * L);
  const float *p = P.part + at * D + d;
  // a thread's first splits are on their way while the factors are made
  constexpr int AHEAD = 8;
  f32x4 v[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; u++) v[u] = *(const f32x4 *)(p + (int64_t)min(x + N * u, P.splits - 1) * stride * D);
  float mk = -__builtin_huge_valf(), lk = 0.0f;
  if ((int)threadIdx.x < 64 && (int)threadIdx.x < P.splits) {
    mk = P.ml[2 * (at + (int64_t)threadIdx.x * stride)];
    lk = P.ml[2 * (at + (int64_t)threadIdx.x * stride) + 1];
  }
  tree_ancestors(t, parent, T);
  const bool live = t.anc[node][0] | t.anc[node][1];
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    float M = mk;
    for (int k = lane + 64; k < P.splits; k += 64) M = fmaxf(M, P.ml[2 * (at + (int64_t)k * stride)]);
    M = dsh_wave_max(M);
    float f = mk == M ? 1.0f : att_exp(mk - M), sum = f * lk;
    s_f[lane] = f;
    for (int k = lane + 64; k < P.splits; k += 64) {
      const float m = P.ml[2 * (at + (int64_t)k * stride)];
      f = m == M ? 1.0f : att_exp(m - M);
      s_f[k] = f;
      sum += f * P.ml[2 * (at + (int64_t)k * stride) + 1];
    }
    sum = dsh_wave_sum(sum);
    const bool none = !live || sum == 0.0f;
    if (lane == 0) {
      s_inv = none ? 0.0f : 1.0f / sum;
      if (A.lse) A.lse[(int64_t)head * T + node] = none ? -__builtin_huge_valf() : M + logf(sum);
    }
  }
  __syncthreads();
  f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  if (x < N) {
#pragma unroll
    for (int u = 0; u < AHEAD; u++)
      if (x + N * u < P.splits) a += s_f[x + N * u] * v[u];
    for (int k = x + N * AHEAD; k < P.splits; k += N) a += s_f[k] * *(const f32x4 *)(p + (int64_t)k * stride * D);
    *(f32x4 *)(s_o[x] + d) = a;
  }
  __syncthreads();
  if ((int)threadIdx.x >= D) return;
  float y = 0.0f;
#pragma unroll
  for (int k = 0; k < N; k++) y += s_o[k][threadIdx.x];
  A.out[node * A.out_stride + (int64_t)head * D + threadIdx.x] = s_inv == 0.0f ? 0.0f : y * s_inv;
}

// ---------------------------------------------------------------------------- verification
// A step's answer hangs on a handful of probabilities and on one row of the vocabulary (one more for every draft that was
// drawn from q and rejected), so what counts is the chain of dependent reads. Every block walks the tree by itself (a wave
// holds a node a lane, twice, with the probabilities at its token fetched ahead), and owns 1/gridDim.x of the row: a sum over
// the row is each block's share, told to all others through tagged words. The last such sum also says which block the drawn
// token lies in, and that block finds it. A chain of 5 or 64 nodes over 129280 tokens 6.3 us, 24 drawn ones 6.3 (one block that did
// it all: 177, 226 and 221); of the kernel's 5.2 us some 1.4 are the probabilities' two round trips, 1.6 the row, 1.8 the sums'
// way from block to block.

// A probability: what is not positive and finite counts as 0.
__device__ __forceinline__ double prob(float x) { return x > 0.0f && x < __builtin_huge_valf() ? (double)x : 0.0; }

struct verify_args {
  int *path, *result;
  const float *p, *q, *u;
  const int *tokens, *parents;
  int64_t p_stride, q_stride;
  int vocab, n, share;  // share: values of a block
  u64 *words;           // [rounds][64][2]
  unsigned epoch;
  int *derr;
};

#define VB 256  // threads; eight consecutive values each at a time
#define VC (8 * VB)
#define VERIFY_TICKS 400000000ull  // of the 100 MHz clock: four seconds

typedef float f32x4_dw __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ double read64(double v, int lane) {
  const u64 x = (u64)__double_as_longlong(v);
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)x, lane), hi = __builtin_amdgcn_readlane((int)(unsigned)(x >> 32), lane);
  return __longlong_as_double((long long)((u64)hi << 32 | lo));
}

struct verify_lds {
  double part[VB / 64], sum[64];
  unsigned gone[VC / 32];
  int fail;
};

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {  // 0 where a lane has no source
  const u64 x = (u64)__double_as_longlong(v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)x, CTRL, 0xF, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(x >> 32), CTRL, 0xF, 0xF, false);
  return __longlong_as_double((long long)((u64)hi << 32 | lo));
}
// Sum over the lanes up to this one; *total: over all.
__device__ __forceinline__ double wave_scan64(double v, double *total) {
  v += dpp64<0x111>(v);  // row_shr:1, 2, 4, 8
  v += dpp64<0x112>(v);
  v += dpp64<0x114>(v);
  v += dpp64<0x118>(v);
  const double r1 = read64(v, 15), r2 = r1 + read64(v, 31), r3 = r2 + read64(v, 47);
  *total = r3 + read64(v, 63);
  const int row = (threadIdx.x >> 4) & 3;
  return row == 0 ? v : (row == 1 ? r1 : row == 2 ? r2 : r3) + v;
}

// What is left of the thread's eight values from v on: max(p - c q, 0), or p without the rejected tokens (bits of gone).
__device__ __forceinline__ void verify_left(double *w, const float *p, const float *q, double c, int v, int end, unsigned gone) {
  float a[8], b[8];
  if (v + 8 <= end) {
    *(f32x4_dw *)a = *(const f32x4_dw *)(p + v);
    *(f32x4_dw *)(a + 4) = *(const f32x4_dw *)(p + v + 4);
    if (q) {
      *(f32x4_dw *)b = *(const f32x4_dw *)(q + v);
      *(f32x4_dw *)(b + 4) = *(const f32x4_dw *)(q + v + 4);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      a[e] = v + e < end ? p[v + e] : 0.0f;
      b[e] = q && v + e < end ? q[v + e] : 0.0f;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; e++) {
    w[e] = prob(a[e]);
    if (q)
      w[e] = fmax(w[e] - c * prob(b[e]), 0.0);
    else if ((gone >> e) & 1)
      w[e] = 0.0;
  }
}

// The rejected tokens among [v0, v0 + VC) as bits: the tokens of the lanes with rej.
__device__ void verify_mark(verify_lds &L, int v0, int tok0, bool rej0, int tok1, bool rej1) {
  __syncthreads();
  if (threadIdx.x < VC / 32) L.gone[threadIdx.x] = 0;
  __syncthreads();
  if (threadIdx.x < 64) {
    const unsigned a = (unsigned)tok0 - (unsigned)v0, b = (unsigned)tok1 - (unsigned)v0;
    if (rej0 && a < VC) atomicOr(&L.gone[a >> 5], 1u << (a & 31));
    if (rej1 && b < VC) atomicOr(&L.gone[b >> 5], 1u << (b & 31));
  }
  __syncthreads();
}

__global__ void __launch_bounds__(VB) k_tree_verify(verify_args A) {
  __shared__ verify_lds L;
  __shared__ int s_path[DSH_TREE_MAX];
  const int n = A.n, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, blocks = gridDim.x, me = blockIdx.x;
  const int lo = me * A.share, hi = min(lo + A.share, A.vocab);  // vocab is 2^30 at most
  // node lane and node lane + 64
  int par0 = -2, par1 = -2, tok0 = -1, tok1 = -1;
  float u0 = 0.0f, u1 = 0.0f;
  double p0 = 0.0, p1 = 0.0, q0 = 0.0, q1 = 0.0;
  if (lane < n) {
    par0 = A.parents[lane];
    tok0 = A.tokens[lane];
    u0 = A.u[lane];
    if (par0 < -1 || par0 >= lane) par0 = -2;
  }
  if (lane + 64 < n) {
    par1 = A.parents[lane + 64];
    tok1 = A.tokens[lane + 64];
    u1 = A.u[lane + 64];
    if (par1 < -1 || par1 >= lane + 64) par1 = -2;
  }
  const float u_last = A.u[n];
  if (par0 > -2 && tok0 >= 0 && tok0 < A.vocab) {
    p0 = prob(A.p[(par0 + 1) * A.p_stride + tok0]);
    if (A.q) q0 = prob(A.q[(par0 + 1) * A.q_stride + tok0]);
  }
  if (par1 > -2 && tok1 >= 0 && tok1 < A.vocab) {
    p1 = prob(A.p[(par1 + 1) * A.p_stride + tok1]);
    if (A.q) q1 = prob(A.q[(par1 + 1) * A.q_stride + tok1]);
  }

  int at = -1, count = 0, rounds = 0;
  double c = 0.0, z = 1.0, spent = 0.0;
  bool summed = false;  // L.sum holds the blocks' shares of what is left at the present context
  // What is left of the row: every block's share in L.sum, their sum; w: the thread's own values of the last piece
  double w[8];
  const auto load = [&](const float *p, const float *q, bool marks, int v0) {
    if (marks) verify_mark(L, v0, tok0, par0 == at, tok1, par1 == at);
    const int v = v0 + 8 * tid;
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = 0.0;
    if (v < hi) verify_left(w, p, q, c, v, hi, marks ? L.gone[tid >> 2] >> (8 * (tid & 3)) : 0);
    return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  };
  const auto row_sum = [&](const float *p, const float *q, bool marks) {
    double mine = 0.0;
    for (int v0 = lo; v0 < hi; v0 += VC) mine += load(p, q, marks, v0);
    wave_scan64(mine, &mine);
    if (lane == 0) L.part[wave] = mine;
    if (tid == 0) L.fail = 0;
    __syncthreads();
    if (wave == 0) {
      mine = ((L.part[0] + L.part[1]) + L.part[2]) + L.part[3];
      u64 *t = A.words + (size_t)rounds * 128;
      const u64 tag = (u64)A.epoch << 32, x = (u64)__double_as_longlong(mine);
      if (blocks > 1 && lane < 2)
        __hip_atomic_store(t + 2 * me + lane, tag | (lane ? x >> 32 : x & 0xFFFFFFFFu), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      double all = lane == me ? mine : 0.0;
      if (blocks > 1) {
        const u64 t0 = __builtin_amdgcn_s_memrealtime();
        bool have = lane >= blocks || lane == me;
        while (!__all(have)) {
          if (!have) {
            const u64 a = __hip_atomic_load(t + 2 * lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const u64 b = __hip_atomic_load(t + 2 * lane + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            have = (a >> 32) == A.epoch && (b >> 32) == A.epoch;
            if (have) all = __longlong_as_double((long long)(b << 32 | (a & 0xFFFFFFFFu)));
          }
          if (__builtin_amdgcn_s_memrealtime() - t0 > VERIFY_TICKS) {
            if (lane == 0) L.fail = 1;
            break;
          }
        }
      }
      L.sum[lane] = all;
    }
    rounds++;
    __syncthreads();
    double s;
    wave_scan64(L.sum[lane], &s);
    summed = true;
    return s;
  };

  u64 m0 = __ballot(par0 == at), m1 = __ballot(par1 == at);
  // a context's first child is tried against p itself: all of those tests at once
  const u64 h0 = __ballot(p0 > 0.0 && (double)u0 * (A.q ? q0 : 1.0) < p0), h1 = __ballot(p1 > 0.0 && (double)u1 * (A.q ? q1 : 1.0) < p1);
  bool failed = false, fresh = true;
  while ((m0 | m1) && !failed) {
    const bool first = m0 != 0;
    const int k = first ? __builtin_ctzll(m0) : __builtin_ctzll(m1);
    if (first)
      m0 &= m0 - 1;
    else
      m1 &= m1 - 1;
    bool hit = ((first ? h0 : h1) >> k) & 1;
    if (!fresh || !hit) {
      const double pk = read64(first ? p0 : p1, k), u = (double)dsh_readlane(first ? u0 : u1, k);
      if (A.q) {
        const double qk = read64(first ? q0 : q1, k), r = fmax(pk - c * qk, 0.0);
        hit = r > 0.0 && u * qk * z < r;
        if (!hit) {
          c += z;
          z = row_sum(A.p + (at + 1) * A.p_stride, A.q + (at + 1) * A.q_stride, false);
          failed = L.fail;
        }
      } else {
        hit = pk > 0.0 && u * (1.0 - spent) < pk;
        if (!hit) {
          spent += pk;
          const int t = __builtin_amdgcn_readlane(first ? tok0 : tok1, k);
          if (par0 == at && tok0 == t) p0 = 0.0;  // nothing is left of the token for the next siblings
          if (par1 == at && tok1 == t) p1 = 0.0;
        }
      }
      fresh = false;
    }
    if (hit) {
      at = first ? k : k + 64;
      if (tid == 0) s_path[count] = at;
      count++;
      c = spent = 0.0;
      z = 1.0;
      summed = false;
      fresh = true;
      m0 = __ballot(par0 == at);
      m1 = __ballot(par1 == at);
    }
  }

  const float *p = A.p + (at + 1) * A.p_stride, *q = A.q && c > 0.0 ? A.q + (at + 1) * A.q_stride : nullptr;
  bool marks = !A.q && __ballot(par0 == at || par1 == at);
  double total = failed ? 0.0 : summed ? z : row_sum(p, q, marks);
  if (!(total > 0.0) && (q || marks) && !failed && !L.fail) {  // nothing is left: p itself
    q = nullptr;
    marks = false;
    total = row_sum(p, q, false);
  }
  failed = failed || (summed && L.fail);
  if (me == 0) {
    __syncthreads();
    if (tid < n) A.path[tid] = tid < count && !failed ? s_path[tid] : -1;
    if (tid == 0) {
      A.result[0] = failed ? 0 : count;
      if (failed || !(total > 0.0)) A.result[1] = -1;
    }
  }
  // any block's: another may have come too late for the others, and then have found all of their sums
  if (failed && tid == 0 && A.derr) __hip_atomic_store(A.derr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  if (failed || !(total > 0.0)) return;
  // the first block whose share crosses the threshold (for a number beyond [0, 1) the last with anything in it), then the
  // wave, the lane and the value
  const double t = (double)u_last * total, share = L.sum[lane];
  double all, before = wave_scan64(share, &all) - share;
  const auto pick = [](u64 crosses, u64 filled) { return crosses ? __builtin_ctzll(crosses) : 63 - __builtin_clzll(filled); };
  if (me != pick(__ballot(share > 0.0 && before + share > t), __ballot(share > 0.0))) return;
  before = read64(before, me);
  int last = -1;
  for (int v0 = lo; v0 < hi; v0 += VC) {
    const double mine = hi - lo > VC ? load(p, q, marks, v0) : ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    double sum, x = wave_scan64(mine, &sum);
    __syncthreads();
    if (lane == 0) L.part[wave] = sum;
    __syncthreads();
    double base = before;
    int own = -1;
#pragma unroll
    for (int k = 0; k < VB / 64; k++) {
      if (k == wave) base = before;
      before += L.part[k];
      if (own < 0 && L.part[k] > 0.0 && before > t) own = k;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (w[e] > 0.0) last = v0 + 8 * tid + e;
    if (own < 0) continue;
    if (own != wave) return;
    const int k = pick(__ballot(mine > 0.0 && base + x > t), __ballot(mine > 0.0));
    if (lane == k) {
      double a = base + (x - mine);
      int token = -1;
      bool done = false;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        a += w[e];
        if (w[e] > 0.0 && !done) {
          token = v0 + 8 * tid + e;
          done = a > t;
        }
      }
      A.result[1] = token;
    }
    return;
  }
  // no more than a rounding is missing (or the number lies beyond [0, 1)): the last value with anything in it
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) last = max(last, __shfl_xor(last, o));
  __syncthreads();
  if (lane == 0) s_path[wave] = last;
  __syncthreads();
  if (tid == 0) A.result[1] = max(max(s_path[0], s_path[1]), max(s_path[2], s_path[3]));
}

// Greedy: one wave, a node a lane, twice.
__global__ void __launch_bounds__(64) k_tree_verify_greedy(int *path, int *result, const int *target, const int *tokens,
                                                           const int *parents, int n) {
  const int lane = threadIdx.x;
  int par0 = -2, par1 = -2, next0 = 0, next1 = 0;
  bool ok0 = false, ok1 = false;
  const int root = target[0];
  if (lane < n) {
    par0 = parents[lane];
    if (par0 < -1 || par0 >= lane) par0 = -2;
    next0 = target[lane + 1];
    ok0 = par0 > -2 && tokens[lane] == target[max(par0, -1) + 1];
  }
  if (lane + 64 < n) {
    par1 = parents[lane + 64];
    if (par1 < -1 || par1 >= lane + 64) par1 = -2;
    next1 = target[lane + 65];
    ok1 = par1 > -2 && tokens[lane + 64] == target[max(par1, -1) + 1];
  }
  int at = -1, count = 0, got0 = -1, got1 = -1;  // got: the path's entries lane and lane + 64
  while (true) {
    const u64 m0 = __ballot(ok0 && par0 == at), m1 = __ballot(ok1 && par1 == at);
    if (!(m0 | m1)) break;
    at = m0 ? __builtin_ctzll(m0) : 64 + __builtin_ctzll(m1);
    if (lane == count) got0 = at;
    if (lane + 64 == count) got1 = at;
    count++;
  }
  if (lane < n) path[lane] = got0;
  if (lane + 64 < n) path[lane + 64] = got1;
  if (lane == 0) result[0] = count;
  const int token = at < 0 ? root : at < 64 ? __builtin_amdgcn_readlane(next0, at) : __builtin_amdgcn_readlane(next1, at & 63);
  if (lane == 0) result[1] = token;
}

// ---------------------------------------------------------------------------- commit
// Blocks (x, head): the columns [256 x, 256 x + 256) of the head's weights, a thread each, eight accepted nodes' scores at a time;
// the last x also the rows that are new, a 16-byte piece of K or V a thread, eight rows at a time in the path's order: a path
// ascends, path[k] >= k, so that a row is read before the one that is written over it where the tree's rows are the cache's own
// from n_cache on. A few KB to a few MB: bound by the launch and by path, score and lse being read one after the other (4
// nodes of 16 over 701 rows 4.2 us, 9 of 64 over 7001 5.6; one score at a time 4.7 and 7.0).
template <int D, bool BF>
__global__ void __launch_bounds__(256) k_tree_commit(dsh_tree_commit_t A) {
  constexpr int P = D / (BF ? 8 : 4);  // pieces of a row
  __shared__ int s_path[DSH_TREE_MAX];
  const int g = blockIdx.y, n = A.n_cache, T = A.n_nodes, claimed = min(max(A.result[0], 0), T);
  const int mine = (int)threadIdx.x < T ? A.path[threadIdx.x] : -1;
  if ((int)threadIdx.x < T) s_path[threadIdx.x] = mine;
  // the path ends before its first entry that is no node
  const u64 stop = __ballot((int)threadIdx.x >= claimed || mine < 0 || mine >= T);
  __shared__ int s_n[4];
  if ((threadIdx.x & 63) == 0) s_n[threadIdx.x >> 6] = stop ? __builtin_ctzll(stop) : 64;
  __syncthreads();
  const int count = s_n[0] < 64 ? s_n[0] : 64 + s_n[1];  // two waves hold every node
  if (A.acc) {
    const int grp = A.n_heads / A.cache.n_heads, j = blockIdx.x * 256 + threadIdx.x;
    if (j < n + count) {
      const int col = j < n ? j : n + s_path[j - n];
      float a = 0.0f;
      for (int h = g * grp; h < (g + 1) * grp; h++)
        for (int k0 = 0; k0 < count; k0 += 8) {
          float s[8], l[8];
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const int64_t row = (int64_t)h * T + s_path[min(k0 + k, count - 1)];
            s[k] = A.scores[row * A.score_stride + col];
            l[k] = A.lse[row];
          }
#pragma unroll
          for (int k = 0; k < 8; k++)
            if (k0 + k < count && l[k] > -__builtin_huge_valf()) a += expf(s[k] - l[k]);
        }
      const int64_t at = g * A.acc_stride + j;
      A.acc_out[at] = j < n ? A.acc[at] + a : a;
    }
  }
  if (blockIdx.x != gridDim.x - 1) return;
  if (A.pos && (int)threadIdx.x < count) A.pos[g * A.pos_stride + n + threadIdx.x] = A.pos0 + threadIdx.x;
  for (int x = threadIdx.x; x < 2 * P; x += 256) {
    constexpr int SZ = BF ? 2 : 4;
    const char *from = (const char *)(x < P ? A.tree.k : A.tree.v) + g * A.tree.head_stride * SZ + 16 * (x < P ? x : x - P);
    char *to = (char *)(x < P ? A.cache.k : A.cache.v) + (g * A.cache.head_stride + n * A.cache.row_stride) * SZ + 16 * (x < P ? x : x - P);
    for (int k0 = 0; k0 < count; k0 += 8) {
      u32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = *(const u32x4 *)(from + s_path[min(k0 + k, count - 1)] * A.tree.row_stride * SZ);
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (k0 + k < count) *(u32x4 *)(to + (k0 + k) * A.cache.row_stride * SZ) = v[k];
    }
  }
}

extern "C" {

#define BY_DIM(D, BF, CASE) \
  switch (D) {              \
    CASE(64, BF)            \
    CASE(128, BF)           \
    CASE(192, BF)           \
    CASE(256, BF)           \
    default:                \
      return hipErrorInvalidValue; \
  }

// The cut of a launch's work, by measurement (10 heads x 128 and an f32 cache, or 16 x 128 over 4 bf16 ones).
// More than one row tile: k_tree_attend_rows (32 nodes over 7001 f32 rows 24.2 us against 24.5, 8 nodes over 4000 bf16 rows 12.8
// against 15.0); one: k_tree_attend, whose four waves share the positions (16 nodes over 7001 rows 20.1 us against 22.0). An
// f32 cache of 192 or 256 dimensions, whose parts do not fit the LDS twice, takes k_tree_attend with up to four row tiles.
// Splits: a block to a CU (one node over 7001 rows: 18.6 us, half as many blocks 20.1, twice as many 20.8; 64 nodes 28.7, 39 and
// 37), but one where that leaves a wave no more than four tiles (5 nodes over 77 rows: 8.4 us; in two splits, joined, 10.7).
static attend_plan attend_cut(const dsh_tree_attn_t *A) {
  attend_plan P;
  memset(&P, 0, sizeof P);
  const int G = A->cache.n_heads, D = A->cache.head_dim;
  const int64_t rows = (int64_t)A->n_nodes * (A->n_heads / G), row_tiles = (rows + 15) / 16;
  P.staged = row_tiles > 1 && (A->cache.bf16 || D <= 128);
  const int AT = A->cache.bf16 || P.staged ? 32 : 16, most = P.staged || D <= 128 ? 8 : 4;
  P.groups = (int)((row_tiles + most - 1) / most);
  P.tile_rows = (int)((row_tiles + P.groups - 1) / P.groups);
  P.pos_waves = P.staged || P.tile_rows > 2 ? 1 : P.tile_rows == 1 ? 4 : 2;
  P.cache_tiles = (int)(((int64_t)A->n_cache + AT - 1) / AT);
  P.tree_tiles = (A->n_nodes + AT - 1) / AT;
  P.gap = P.cache_tiles;
  // R-SWA: no node sees what lies between the reference positions and the first root's window
  if (A->window > 0 && !A->scores && A->n_cache >= A->prefill_len) {
    const int64_t lo = (int64_t)A->n_cache + 1 - A->window;
    const int from = (int)(((int64_t)A->prefill_len + AT - 1) / AT), to = lo > 0 ? (int)(lo / AT) : 0;
    if (to > from) {
      P.gap = from;
      P.skip = to - from;
    }
  }
  const int64_t tiles = (int64_t)P.cache_tiles - P.skip + P.tree_tiles;
  const int64_t want = 256 / ((int64_t)G * P.groups);
  int64_t splits = (tiles + P.pos_waves - 1) / P.pos_waves;
  if (splits <= 4) splits = 1;
  if (splits > want) splits = want;
  if (splits > 1024) splits = 1024;
  if (splits < 1) splits = 1;
  P.per = (int)((tiles + splits - 1) / splits);
  P.splits = (int)((tiles + P.per - 1) / P.per);
  P.grp = A->n_heads / G;
  P.inv_nodes = 1.0f / (float)A->n_nodes;
  return P;
}

// Floats of workspace for the splits' sums.
size_t dsh_tree_attention_work(const dsh_tree_attn_t *A) {
  const attend_plan P = attend_cut(A);
  if (P.splits == 1) return 0;
  return (size_t)A->cache.n_heads * P.groups * P.splits * 16 * P.tile_rows * (A->cache.head_dim + 2);
}

hipError_t dsh_launch_tree_attention(const dsh_tree_attn_t *A, float *work, hipStream_t s) {
  if (A->n_nodes < 1 || A->n_nodes > DSH_TREE_MAX) return hipErrorInvalidValue;
  attend_plan P = attend_cut(A);
  const int D = A->cache.head_dim, W = P.tile_rows * P.pos_waves;
  if (W > 8 || (!P.staged && W > 4) || P.groups > 65535 || (P.splits > 1 && !work)) return hipErrorInvalidValue;
  P.part = work;
  P.ml = work ? work + (size_t)A->cache.n_heads * P.groups * P.splits * 16 * P.tile_rows * D : nullptr;
  const dim3 grid(P.splits, A->cache.n_heads, P.groups);
  const size_t lds = P.pos_waves > 1 ? (size_t)W * 16 * ((D < 128 ? D : 128) + 4) * 4 : 0;
#define CASE(D, BF)                                                                   \
  case D:                                                                             \
    if (P.staged) {                                                                   \
      if constexpr (BF || D <= 128) {                                                 \
        if (P.tile_rows <= 4)                                                         \
          k_tree_attend_rows<D, BF, 4><<<grid, 512, 0, s>>>(*A, P);                   \
        else if constexpr (BF) {                                                      \
          if (P.tile_rows <= 6)                                                       \
            k_tree_attend_rows<D, BF, 2><<<grid, 512, 0, s>>>(*A, P);                 \
          else                                                                        \
            k_tree_attend_rows<D, BF, 8><<<grid, 512, 0, s>>>(*A, P);                 \
        } else                                                                        \
          k_tree_attend_rows<D, BF, 8><<<grid, 512, 0, s>>>(*A, P);                   \
      }                                                                               \
    } else {                                                                          \
      k_tree_attend<D, BF><<<grid, 64 * W, lds, s>>>(*A, P);                          \
    }                                                                                 \
    if (P.splits > 1)                                                                 \
      k_tree_join<D><<<dim3(A->n_nodes * (A->n_heads / A->cache.n_heads), A->cache.n_heads), 256, 0, s>>>(*A, P); \
    break;
  if (A->cache.bf16) {
    BY_DIM(D, true, CASE)
  } else {
    BY_DIM(D, false, CASE)
  }
#undef CASE
  return hipGetLastError();
}

hipError_t dsh_launch_tree_verify(int *path, int *result, const float *p, int64_t p_stride, const float *q,
                                  int64_t q_stride, int vocab, const int *tokens, const int *parents, int n_nodes,
                                  const float *u, unsigned long long *words, unsigned epoch, int *derr, hipStream_t s) {
  if (n_nodes < 0 || n_nodes > DSH_TREE_MAX || vocab < 1) return hipErrorInvalidValue;
  // a block per VC values, 64 at most (a lane each when the shares are told); shares in whole eights
  const int want = (int)(((int64_t)vocab + VC - 1) / VC), blocks = want < 64 ? want : 64;
  const int64_t share = (((int64_t)vocab + blocks - 1) / blocks + 7) / 8 * 8;
  const verify_args a{path, result, p, q, u, tokens, parents, p_stride, q_stride, vocab, n_nodes, (int)share, words, epoch, derr};
  k_tree_verify<<<(int)((vocab + share - 1) / share), VB, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t dsh_launch_tree_verify_greedy(int *path, int *result, const int *target, const int *tokens, const int *parents,
                                         int n_nodes, hipStream_t s) {
  if (n_nodes < 0 || n_nodes > DSH_TREE_MAX) return hipErrorInvalidValue;
  k_tree_verify_greedy<<<1, 64, 0, s>>>(path, result, target, tokens, parents, n_nodes);
  return hipGetLastError();
}

hipError_t dsh_launch_tree_commit(const dsh_tree_commit_t *A, hipStream_t s) {
  if (A->n_nodes < 1 || A->n_nodes > DSH_TREE_MAX) return hipErrorInvalidValue;
  const dim3 g(A->acc ? (A->n_cache + A->n_nodes + 255) / 256 : 1, A->cache.n_heads);
#define CASE(D, BF)                             \
  case D:                                       \
    k_tree_commit<D, BF><<<g, 256, 0, s>>>(*A); \
    break;
  if (A->cache.bf16) {
    BY_DIM(A->cache.head_dim, true, CASE)
  } else {
    BY_DIM(A->cache.head_dim, false, CASE)
  }
#undef CASE
  return hipGetLastError();
}

}  // extern "C"
