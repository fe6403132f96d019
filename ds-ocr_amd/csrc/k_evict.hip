// k_evict.hip — which rows of a KV cache stay (k_kv_select: per head the rows with the least attention weight go), and the
// moves that bring them together (k_kv_move).
#include "dsh.h"
#include "k_core.h"

#define ET 1024
#define EW (ET / 64)
#define EVICT_OWN 131072  // bytes of K and V rows of a head

typedef unsigned long long u64;

// Floats in ascending order as unsigned numbers; -0 as 0, a NaN as -inf.
__device__ __forceinline__ uint32_t evict_key(float a) {
  if (a != a) a = -__builtin_huge_valf();
  const uint32_t u = __float_as_uint(a + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A row of a head as a number: `gone` = n - keep rows with the lowest numbers go, the lower row first among equal ones. Where
// there are unguarded rows enough, a guarded row is above all; where not, an unguarded one is below all.
__device__ __forceinline__ uint32_t evict_number(float a, bool guarded, bool spill) {
  return guarded == spill ? evict_key(a) : spill ? 0u : 0xFFFFFFFFu;
}

// Sum over the block of three counts (each a wave's, the same in all its lanes), by way of s (3 x EW words, not in use by
// the call before this one).
__device__ __forceinline__ void evict_sums(int (*s)[EW], int &a, int &b, int &c) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane < 3) s[lane][wave] = lane == 0 ? a : lane == 1 ? b : c;
  __syncthreads();
  int x = lane < 48 ? s[lane >> 4][lane & 15] : 0;
  x += __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false);   // over the 16 lanes of a row
  x += __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x140, 0xF, 0xF, false);
  a = __builtin_amdgcn_readlane(x, 0);
  b = __builtin_amdgcn_readlane(x, 16);
  c = __builtin_amdgcn_readlane(x, 32);
}

struct evict_lds {
  int cnt[2][3][EW];
  uint32_t few[64], T;
  int n_few, left, equal;
};

// The gone-th lowest number T, two bits at a step: each counts the numbers below three candidates by wave votes (count(t...)
// adds a wave's), which costs the same whatever the numbers are; a histogram in LDS piles up on the few exponents that
// weights have. Once at most 64 numbers are in question, gather(T, mask) puts them in few, and one wave ranks them. left: how
// many of those equal to T go, equal: of how many.
template <typename F, typename G>
__device__ __forceinline__ void evict_threshold(evict_lds &L, int gone, int n, uint32_t &T, int &left, int &equal, F count,
                                                G gather) {
  T = 0;
  left = equal = 0;  // no number is 0 unless it goes
  if (gone == 0) return;
  if (threadIdx.x == 0) L.n_few = 0;
  int under = 0, over = n;  // numbers below T, and below T + 4^k
  for (int shift = 30; shift >= 0; shift -= 2) {
    const uint32_t t1 = T | 1u << shift, t2 = T | 2u << shift, t3 = T | 3u << shift;
    int c1 = 0, c2 = 0, c3 = 0;
    count(t1, t2, t3, c1, c2, c3);
    evict_sums(L.cnt[(shift >> 1) & 1], c1, c2, c3);
    if (c3 < gone) {
      T = t3;
      under = c3;
    } else if (c2 < gone) {
      T = t2;
      under = c2;
      over = c3;
    } else if (c1 < gone) {
      T = t1;
      under = c1;
      over = c2;
    } else {
      over = c1;
    }
    if (shift > 0 && over - under <= 64) {
      gather(T, ~0u << shift);
      __syncthreads();
      if (threadIdx.x < 64) {
        const int lane = threadIdx.x, m = over - under;
        const uint32_t k = lane < m ? L.few[lane] : 0xFFFFFFFFu;
        int less = 0, leq = 0;
        for (int x = 0; x < m; x++) {
          const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)k, x);
          less += o < k;
          leq += o <= k;
        }
        if (lane < m && under + less < gone && under + leq >= gone) {  // equal lanes write the same
          L.T = k;
          L.left = gone - under - less;
          L.equal = leq - less;
        }
      }
      __syncthreads();
      T = L.T;
      left = L.left;
      equal = L.equal;
      return;
    }
  }
  left = gone - under;
  equal = over - under;
}

// Exclusive prefix of N cells (a multiple of 64) by one wave; s[N] becomes the sum.
template <int N>
__device__ __forceinline__ void evict_prefix(int *s) {
  constexpr int P = N / 64;
  const int lane = threadIdx.x & 63;
  int v[P], sum = 0;
#pragma unroll
  for (int k = 0; k < P; k++) {
    v[k] = s[P * lane + k];
    sum += v[k];
  }
  int x = sum;
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  const int r0 = __builtin_amdgcn_readlane(x, 15), r1 = r0 + __builtin_amdgcn_readlane(x, 31);
  const int r2 = r1 + __builtin_amdgcn_readlane(x, 47);
  x += lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r1 : r2;
  if (lane == 63) s[N] = x;
  x -= sum;
#pragma unroll
  for (int k = 0; k < P; k++) {
    s[P * lane + k] = x;
    x += v[k];
  }
}

// K and V rows of the movers into the holes, 16 bytes a thread, four pieces under way. P: 16-byte pieces of a row.
__device__ __forceinline__ void evict_move(const dsh_kv_evict_t &A, int h, int count, const int *hole, const int *mover, int P,
                                           int64_t first, int64_t step) {
  const int64_t rs = A.cache.row_stride * (A.cache.bf16 ? 2 : 4), hs = A.cache.head_stride * (A.cache.bf16 ? 2 : 4);
  char *k = (char *)A.cache.k + h * hs, *v = (char *)A.cache.v + h * hs;
  const int64_t total = (int64_t)count * 2 * P;
  for (int64_t x = first; x < total; x += 4 * step) {
    u32x4 y[4];
    char *to[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int64_t i = x + u * step;
      to[u] = nullptr;
      if (i < total) {
        const int r = (int)((uint64_t)i / (unsigned)(2 * P)), piece = (int)(i - (int64_t)r * 2 * P);
        char *b = piece < P ? k + 16 * piece : v + 16 * (piece - P);
        to[u] = b + hole[r] * rs;
        y[u] = *(const u32x4 *)(b + mover[r] * rs);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (to[u]) *(u32x4 *)to[u] = y[u];
  }
}

// One block per head, up to 1024 E rows in registers; thread t has the rows 1024 e + t. Ranks (among the equal numbers, then of
// the holes below `keep` and of the rows that fill them) come from votes too: a count for every 64 rows, a prefix over those.
// Workspace: per head a count, then holes [most] and movers [most], most = min(n - keep, keep).
// move: the rows' own pieces, where the block itself moves them (0: k_kv_move does).
template <int E>
__global__ void __launch_bounds__(ET) k_kv_select(dsh_kv_evict_t A, int most, int move) {
  constexpr int N = E * EW;
  __shared__ evict_lds L;
  __shared__ int s_a[N + 1], s_b[N + 1];
  extern __shared__ uint16_t s_mv[];  // [most]
  const int h = blockIdx.x, n = A.n, keep = A.keep, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float *acc = A.acc + h * A.acc_stride;
  const int *pos = A.pos ? A.pos + h * A.pos_stride : nullptr;
  int *count = A.work + h, *hole = A.work + A.cache.n_heads + (int64_t)h * 2 * most, *mover = hole + most;
  const u64 below = (1ull << lane) - 1;
  uint32_t key[E];
  int p[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = ET * e + tid;
    key[e] = __float_as_uint(j < n ? acc[j] : 0.0f);
    p[e] = j < n && pos ? pos[j] : j;
  }
  uint32_t guard = 0;
  int free_rows = 0, none = 0, none2 = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const bool g = p[e] < A.sink || p[e] >= A.recent_from;
    guard |= (uint32_t)g << e;
    free_rows += __popcll(__ballot(ET * e + tid < n && !g));
  }
  evict_sums(L.cnt[0], free_rows, none, none2);  // the first step takes the other
  const int gone = n - keep;
  const bool spill = gone > free_rows;
#pragma unroll
  for (int e = 0; e < E; e++)
    key[e] = ET * e + tid < n ? evict_number(__uint_as_float(key[e]), (guard >> e) & 1, spill) : 0xFFFFFFFFu;
  uint32_t T;
  int left, equal;
  const auto count_below = [&](uint32_t t1, uint32_t t2, uint32_t t3, int &c1, int &c2, int &c3) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      c1 += __popcll(__ballot(key[e] < t1));
      c2 += __popcll(__ballot(key[e] < t2));
      c3 += __popcll(__ballot(key[e] < t3));
    }
  };
  evict_threshold(L, gone, n, T, left, equal, count_below, [&](uint32_t t, uint32_t mask) {
#pragma unroll
    for (int e = 0; e < E; e++)
      if (ET * e + tid < n && (key[e] & mask) == t) L.few[atomicAdd(&L.n_few, 1) & 63] = key[e];
  });
  uint32_t stays = 0;
  if (left == equal) {
#pragma unroll
    for (int e = 0; e < E; e++) stays |= (uint32_t)(ET * e + tid < n && key[e] > T) << e;
  } else {  // ranks among the equal ones
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int c = __popcll(__ballot(key[e] == T));
      if (lane == 0) s_a[e * EW + wave] = c;
    }
    __syncthreads();
    if (wave == 0) evict_prefix<N>(s_a);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int rank = s_a[e * EW + wave] + __popcll(__ballot(key[e] == T) & below);
      stays |= (uint32_t)(ET * e + tid < n && (key[e] > T || (key[e] == T && rank >= left))) << e;
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = ET * e + tid;
    const bool s = (stays >> e) & 1;
    const int ch = __popcll(__ballot(j < keep && !s)), cm = __popcll(__ballot(j >= keep && s));
    if (lane == 0) {
      s_a[e * EW + wave] = ch;
      s_b[e * EW + wave] = cm;
    }
  }
  __syncthreads();
  if (wave == 0) evict_prefix<N>(s_a);
  if (wave == 1) evict_prefix<N>(s_b);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = ET * e + tid;
    const bool m = j >= keep && ((stays >> e) & 1);
    const int r = s_b[e * EW + wave] + __popcll(__ballot(m) & below);
    if (m) {
      s_mv[r] = (uint16_t)j;
      mover[r] = j;
    }
  }
  if (tid == 0) *count = s_a[N];
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = ET * e + tid;
    const bool o = j < keep && !((stays >> e) & 1);
    const int r = s_a[e * EW + wave] + __popcll(__ballot(o) & below);
    if (o) hole[r] = j;
    if (j < keep) {
      const int from = o ? s_mv[r] : j;
      if (A.slots) A.slots[(int64_t)h * keep + j] = from;
      if (A.acc_out) A.acc_out[h * A.acc_out_stride + j] = acc[from];
      if (A.pos_out) A.pos_out[h * A.pos_out_stride + j] = pos[from];
    }
  }
  if (move) {
    __syncthreads();
    evict_move(A, h, s_a[N], hole, mover, move, tid, ET);
  }
}

// The same for more rows than that, read again at every step; a thread's rows are consecutive where ranks are counted.
__global__ void __launch_bounds__(ET) k_kv_select_long(dsh_kv_evict_t A, int most) {
  __shared__ evict_lds L;
  __shared__ int s_a[ET + 1], s_b[ET + 1];
  const int h = blockIdx.x, n = A.n, keep = A.keep, tid = threadIdx.x;
  const float *acc = A.acc + h * A.acc_stride;
  const int *pos = A.pos ? A.pos + h * A.pos_stride : nullptr;
  int *count = A.work + h, *hole = A.work + A.cache.n_heads + (int64_t)h * 2 * most, *mover = hole + most;
  const auto guarded = [&](int j) {
    const int p = pos ? pos[j] : j;
    return p < A.sink || p >= A.recent_from;
  };
  int free_rows = 0, none = 0, none2 = 0;
  for (int j0 = 0; j0 < n; j0 += ET) free_rows += __popcll(__ballot(j0 + tid < n && !guarded(min(j0 + tid, n - 1))));
  evict_sums(L.cnt[0], free_rows, none, none2);  // the first step takes the other
  const int gone = n - keep;
  const bool spill = gone > free_rows;
  const auto number = [&](int j) { return evict_number(acc[j], guarded(j), spill); };
  uint32_t T;
  int left, equal;
  const auto count_below = [&](uint32_t t1, uint32_t t2, uint32_t t3, int &c1, int &c2, int &c3) {
    for (int j0 = 0; j0 < n; j0 += ET) {
      const uint32_t k = j0 + tid < n ? number(j0 + tid) : 0xFFFFFFFFu;
      c1 += __popcll(__ballot(k < t1));
      c2 += __popcll(__ballot(k < t2));
      c3 += __popcll(__ballot(k < t3));
    }
  };
  evict_threshold(L, gone, n, T, left, equal, count_below, [&](uint32_t t, uint32_t mask) {
    for (int j = tid; j < n; j += ET) {
      const uint32_t k = number(j);
      if ((k & mask) == t) L.few[atomicAdd(&L.n_few, 1) & 63] = k;
    }
  });
  const int per = (int)(((int64_t)n + ET - 1) / ET);
  const int j0 = (int)min((int64_t)tid * per, (int64_t)n), j1 = (int)min((int64_t)j0 + per, (int64_t)n);
  int ties = 0;
  for (int j = j0; j < j1; j++) ties += number(j) == T;
  s_a[tid] = ties;
  __syncthreads();
  if (tid < 64) evict_prefix<ET>(s_a);
  __syncthreads();
  const int tie0 = s_a[tid];
  const auto stays = [&](int j, int &tie) {
    const uint32_t k = number(j);
    return k > T || (k == T && tie++ >= left);
  };
  int holes = 0, movers = 0, tie = tie0;
  for (int j = j0; j < j1; j++) {
    const bool s = stays(j, tie);
    holes += j < keep && !s;
    movers += j >= keep && s;
  }
  __syncthreads();
  s_a[tid] = holes;
  s_b[tid] = movers;
  __syncthreads();
  if (tid < 64)
    evict_prefix<ET>(s_a);
  else if (tid < 128)
    evict_prefix<ET>(s_b);
  __syncthreads();
  int oh = s_a[tid], om = s_b[tid];
  tie = tie0;
  for (int j = j0; j < j1; j++) {
    const bool s = stays(j, tie);
    if (j < keep && !s) hole[oh++] = j;
    if (j >= keep && s) mover[om++] = j;
  }
  const int moves = s_a[ET];
  if (tid == 0) *count = moves;
  __syncthreads();
  // the rows that stay where they are (all of them first), then the holes
  for (int j = tid; j < keep; j += ET) {
    if (A.slots) A.slots[(int64_t)h * keep + j] = j;
    if (A.acc_out && A.acc_out != A.acc) A.acc_out[h * A.acc_out_stride + j] = acc[j];
    if (A.pos_out && A.pos_out != A.pos) A.pos_out[h * A.pos_out_stride + j] = pos[j];
  }
  __syncthreads();
  for (int r = tid; r < moves; r += ET) {
    const int j = hole[r], from = mover[r];
    if (A.slots) A.slots[(int64_t)h * keep + j] = from;
    if (A.acc_out) A.acc_out[h * A.acc_out_stride + j] = acc[from];
    if (A.pos_out) A.pos_out[h * A.pos_out_stride + j] = pos[from];
  }
}

template <int P>
__global__ void __launch_bounds__(256) k_kv_move(dsh_kv_evict_t A, int most) {
  const int h = blockIdx.y;
  const int *hole = A.work + A.cache.n_heads + (int64_t)h * 2 * most;
  evict_move(A, h, A.work[h], hole, hole + most, P, blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

extern "C" {

static int evict_most(int n, int keep) { return n - keep < keep ? n - keep : keep; }

size_t dsh_kv_evict_work(int n_heads, int n, int keep) { return (size_t)n_heads * (1 + 2 * (size_t)evict_most(n, keep)); }

hipError_t dsh_launch_kv_evict(const dsh_kv_evict_t *A, hipStream_t s) {
  const int most = evict_most(A->n, A->keep), G = A->cache.n_heads;
  const size_t lds = (size_t)(most + 1) * 2;  // 32 KB at most
  const int pieces = A->cache.head_dim / (A->cache.bf16 ? 8 : 4);
  // few rows are moved by the block that chose them
  const int move = A->n <= 32 * ET && (int64_t)most * 32 * pieces <= EVICT_OWN ? pieces : 0;
  if (A->n <= 4 * ET)
    k_kv_select<4><<<G, ET, lds, s>>>(*A, most, move);
  else if (A->n <= 8 * ET)
    k_kv_select<8><<<G, ET, lds, s>>>(*A, most, move);
  else if (A->n <= 16 * ET)
    k_kv_select<16><<<G, ET, lds, s>>>(*A, most, move);
  else if (A->n <= 32 * ET)
    k_kv_select<32><<<G, ET, lds, s>>>(*A, most, move);
  else
    k_kv_select_long<<<G, ET, 0, s>>>(*A, most);
  if (most == 0 || move) return hipGetLastError();
  const int64_t want = ((int64_t)most * 2 * pieces + 1023) / 1024, cap = G < 2048 ? 2048 / G : 1;
  const dim3 g((unsigned)(want < cap ? want : cap), G);
#define MV(N)                                      \
  case N:                                          \
    k_kv_move<N><<<g, 256, 0, s>>>(*A, most);      \
    break;
  switch (pieces) {
    MV(8) MV(16) MV(24) MV(32) MV(48) MV(64)
    default:
      return hipErrorInvalidValue;
  }
#undef MV
  return hipGetLastError();
}

}  // extern "C"
