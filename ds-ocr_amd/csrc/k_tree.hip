// k_tree.hip — drafted tokens over a KV cache: attention of a tree's nodes (k_tree_attend), verification of the drafts
// (k_tree_verify), and the accepted nodes' rows and weights into the cache (k_tree_commit).
#include "dsh.h"
#include "k_core.h"

typedef unsigned long long u64;

// ---------------------------------------------------------------------------- the tree
// Every node's ancestors-or-self as 128 bits and its depth, from the parents, by pointer doubling: after round r a node
// knows its next 2^r ancestors, so that a chain of 128 takes 7 rounds. A padding node (a parent outside [-1, i), or a padding
// node above it) has no bits. Called by every thread of a block of at least DSH_TREE_MAX.
struct tree_lds {
  u64 anc[DSH_TREE_MAX][2];
  int up[DSH_TREE_MAX];
};
__device__ void tree_ancestors(tree_lds &t, const int *parents, int n) {
  const int i = threadIdx.x;
  u64 lo = 0, hi = 0;
  int up = -2;
  if (i < n) {
    up = parents[i];
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
__device__ __forceinline__ bool tree_bit(const u64 *anc, int a) { return (anc[a >> 6] >> (a & 63)) & 1; }
__device__ __forceinline__ int tree_depth(const u64 *anc) { return __popcll(anc[0]) + __popcll(anc[1]) - 1; }

// Whether a node at position pos sees position p (what it sees at all): R-SWA's reference positions and window.
__device__ __forceinline__ bool tree_in_window(int p, int pos, int prefill_len, int window) {
  return window <= 0 || pos < prefill_len || p < prefill_len || p > pos - window;
}

// ---------------------------------------------------------------------------- attention
template <bool BF>
__device__ __forceinline__ float kv_at(const void *p, int64_t i) {
  return BF ? dsh_bf16_to_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}

// One block per node and query head: every wave runs the softmax over its share of the positions with a running maximum
// and sum, the lanes over the head's dimensions, and the waves' results are put together at the end.
template <int D, bool BF>
__global__ void __launch_bounds__(256) k_tree_attend(dsh_tree_attn_t A) {
  constexpr int E = D / 64;
  __shared__ tree_lds t;
  __shared__ float s_o[4][D], s_m[4], s_l[4];
  const int i = blockIdx.x, h = blockIdx.y, kh = h / (A.n_heads / A.cache.n_heads);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  tree_ancestors(t, A.parents, A.n_nodes);
  const bool live = t.anc[i][0] | t.anc[i][1];
  const int pos = A.n_cache + tree_depth(t.anc[i]);
  float q[E], o[E], m = -__builtin_huge_valf(), l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; e++) {
    q[e] = A.q[i * A.q_stride + (int64_t)h * D + lane + 64 * e];
    o[e] = 0.0f;
  }
  float *sc = A.scores ? A.scores + ((int64_t)h * A.n_nodes + i) * A.score_stride : nullptr;
  for (int j = wave; j < A.n_cache + A.n_nodes; j += 4) {
    const bool own = j >= A.n_cache;
    const int a = j - A.n_cache;
    bool see = live && (!own || tree_bit(t.anc[i], a));
    see = see && tree_in_window(own ? A.n_cache + tree_depth(t.anc[a]) : j, pos, A.prefill_len, A.window);
    float s = -__builtin_huge_valf();
    if (see) {
      const dsh_kv_t &c = own ? A.tree : A.cache;
      const int64_t at = (own ? a : j) * c.row_stride + kh * c.head_stride;
      float d = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e++) d = __builtin_fmaf(q[e], kv_at<BF>(c.k, at + lane + 64 * e), d);
      s = dsh_wave_sum(d) * A.scale;
      const float mn = fmaxf(m, s), f = mn == m ? 1.0f : expf(m - mn), w = mn == s ? 1.0f : expf(s - mn);
      l = l * f + w;
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = o[e] * f + w * kv_at<BF>(c.v, at + lane + 64 * e);
      m = mn;
    }
    if (sc && lane == 0) sc[j] = s;
  }
#pragma unroll
  for (int e = 0; e < E; e++) s_o[wave][lane + 64 * e] = o[e];
  if (lane == 0) {
    s_m[wave] = m;
    s_l[wave] = l;
  }
  __syncthreads();
  const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float f[4], L = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    f[w] = s_m[w] == M ? 1.0f : expf(s_m[w] - M);
    L += f[w] * s_l[w];
  }
  for (int d = threadIdx.x; d < D; d += 256) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) v += f[w] * s_o[w][d];
    A.out[i * A.out_stride + (int64_t)h * D + d] = L == 0.0f ? 0.0f : v / L;
  }
  if (A.lse && threadIdx.x == 0) A.lse[(int64_t)h * A.n_nodes + i] = L == 0.0f ? -__builtin_huge_valf() : M + logf(L);
}

// ---------------------------------------------------------------------------- verification
// A probability: what is not positive and finite counts as 0.
__device__ __forceinline__ double prob(float x) { return x > 0.0f && x < __builtin_huge_valf() ? (double)x : 0.0; }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

struct verify_args {
  int *path, *result;
  const float *p, *q, *u;
  const int *target, *tokens, *parents;
  int64_t p_stride, q_stride;
  int vocab, n;
};

// What is left of a context's distribution: max(p - c q, 0), or p without the rejected tokens.
struct residual {
  const float *p, *q;
  double c;
  const int *gone;  // LDS
  int n_gone;
  __device__ __forceinline__ double at(int v) const {
    const double x = prob(p[v]);
    if (q) return fmax(x - c * prob(q[v]), 0.0);
    for (int k = 0; k < n_gone; k++)
      if (gone[k] == v) return 0.0;
    return x;
  }
};

#define VT 1024
// Sum of the residual over [lo, hi) (every thread gets it).
__device__ double residual_sum(const residual &r, int lo, int hi, double *s_w) {
  double a = 0.0;
  for (int v = lo + threadIdx.x; v < hi; v += VT) a += r.at(v);
  a = wave_sum64(a);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_w[threadIdx.x >> 6] = a;
  __syncthreads();
  a = 0.0;
  for (int w = 0; w < VT / 64; w++) a += s_w[w];
  return a;
}

// One block: the walk (every thread the same), and the draw from what is left.
__global__ void __launch_bounds__(VT) k_tree_verify(verify_args A) {
  __shared__ int s_par[DSH_TREE_MAX], s_tok[DSH_TREE_MAX], s_gone[DSH_TREE_MAX];
  __shared__ double s_w[VT / 64];
  const int n = A.n, tid = threadIdx.x;
  if (tid < n) {
    s_par[tid] = A.parents[tid];
    s_tok[tid] = A.tokens[tid];
    A.path[tid] = -1;
  }
  __syncthreads();
  int at = -1, count = 0, n_gone = 0;
  double c = 0.0, z = 1.0, spent = 0.0;
  for (int k = 0; k < n; k++) {  // children come after their parents
    if (s_par[k] != at) continue;
    const int tok = s_tok[k];
    bool hit;
    if (A.target) {
      hit = tok == A.target[at + 1];
    } else if (tok < 0 || tok >= A.vocab) {
      hit = false;
      if (A.q) {
        c += z;
        z = residual_sum(residual{A.p + (at + 1) * A.p_stride, A.q + (at + 1) * A.q_stride, c, s_gone, 0}, 0, A.vocab, s_w);
      }
    } else {
      const float *p = A.p + (at + 1) * A.p_stride;
      const double u = (double)A.u[k];
      if (A.q) {
        const float *q = A.q + (at + 1) * A.q_stride;
        const double qt = prob(q[tok]), r = fmax(prob(p[tok]) - c * qt, 0.0);
        hit = r > 0.0 && u * qt * z < r;
        if (!hit) {
          c += z;
          z = residual_sum(residual{p, q, c, s_gone, 0}, 0, A.vocab, s_w);
        }
      } else {
        double r = prob(p[tok]);
        for (int g = 0; g < n_gone; g++)
          if (s_gone[g] == tok) r = 0.0;
        hit = r > 0.0 && u * (1.0 - spent) < r;
        if (!hit) {
          __syncthreads();
          if (tid == 0) s_gone[n_gone] = tok;
          __syncthreads();
          n_gone++;
          spent += r;
        }
      }
    }
    if (hit) {
      if (tid == 0) A.path[count] = k;
      count++;
      at = k;
      n_gone = 0;
      c = 0.0;
      z = 1.0;
      spent = 0.0;
    }
  }
  if (tid == 0) A.result[0] = count;
  if (A.target) {
    if (tid == 0) A.result[1] = A.target[at + 1];
    return;
  }
  residual r{A.p + (at + 1) * A.p_stride, A.q ? A.q + (at + 1) * A.q_stride : nullptr, c, s_gone, n_gone};
  double total = residual_sum(r, 0, A.vocab, s_w);
  if (!(total > 0.0)) {
    r.q = nullptr;
    r.n_gone = 0;
    total = residual_sum(r, 0, A.vocab, s_w);
  }
  if (!(total > 0.0)) {
    if (tid == 0) A.result[1] = -1;
    return;
  }
  // the piece of VT values that the threshold falls in, then the value
  const double t = (double)A.u[n] * total;
  double cum = 0.0;
  int last = -1;  // the last piece with anything in it
  for (int lo = 0; lo < A.vocab; lo += VT) {
    const double s = residual_sum(r, lo, min(lo + VT, A.vocab), s_w);
    if (s > 0.0) last = lo;
    if (s > 0.0 && cum + s > t) break;
    if (lo + VT < A.vocab) cum += s;
  }
  if (tid == 0) {
    double a = cum;
    int pick = -1;
    for (int v = last; v < min(last + VT, A.vocab); v++) {
      const double w = r.at(v);
      if (!(w > 0.0)) continue;
      pick = v;
      a += w;
      if (a > t) break;
    }
    A.result[1] = pick;
  }
}

// ---------------------------------------------------------------------------- commit
// Blocks (x, head): the columns [256 x, 256 x + 256) of the head's weights; the last x the rows that are new.
template <int D, typename T>
__global__ void __launch_bounds__(256) k_tree_commit(dsh_tree_commit_t A) {
  __shared__ int s_path[DSH_TREE_MAX], s_n;
  const int g = blockIdx.y, n = A.n_cache, grp = A.n_heads / (A.acc ? A.cache.n_heads : 1);
  if (threadIdx.x == 0) s_n = min(max(A.result[0], 0), A.n_nodes);
  __syncthreads();
  if ((int)threadIdx.x < A.n_nodes) s_path[threadIdx.x] = A.path[threadIdx.x];
  __syncthreads();
  int count = 0;
  while (count < s_n && s_path[count] >= 0 && s_path[count] < A.n_nodes) count++;
  if (A.acc) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j < n + count) {
      const int col = j < n ? j : n + s_path[j - n];
      float a = 0.0f;
      for (int h = g * grp; h < (g + 1) * grp; h++)
        for (int k = 0; k < count; k++) {
          const int64_t row = (int64_t)h * A.n_nodes + s_path[k];
          const float l = A.lse[row];
          if (l > -__builtin_huge_valf()) a += expf(A.scores[row * A.score_stride + col] - l);
        }
      const int64_t at = g * A.acc_stride + j;
      A.acc_out[at] = j < n ? A.acc[at] + a : a;
    }
  }
  if (blockIdx.x != gridDim.x - 1) return;
  if (A.pos && (int)threadIdx.x < count) A.pos[g * A.pos_stride + n + threadIdx.x] = A.pos0 + threadIdx.x;
  for (int x = threadIdx.x; x < count * D; x += 256) {
    const int k = x / D, d = x - k * D;
    const int64_t from = s_path[k] * A.tree.row_stride + g * A.tree.head_stride + d;
    const int64_t to = (int64_t)(n + k) * A.cache.row_stride + g * A.cache.head_stride + d;
    ((T *)A.cache.k)[to] = ((const T *)A.tree.k)[from];
    ((T *)A.cache.v)[to] = ((const T *)A.tree.v)[from];
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

hipError_t dsh_launch_tree_attention(const dsh_tree_attn_t *A, hipStream_t s) {
  if (A->n_nodes < 1 || A->n_nodes > DSH_TREE_MAX) return hipErrorInvalidValue;
  const dim3 g(A->n_nodes, A->n_heads);
#define CASE(D, BF)                         \
  case D:                                   \
    k_tree_attend<D, BF><<<g, 256, 0, s>>>(*A); \
    break;
  if (A->cache.bf16) {
    BY_DIM(A->cache.head_dim, true, CASE)
  } else {
    BY_DIM(A->cache.head_dim, false, CASE)
  }
#undef CASE
  return hipGetLastError();
}

hipError_t dsh_launch_tree_verify(int *path, int *result, const float *p, int64_t p_stride, const float *q,
                                  int64_t q_stride, int vocab, const int *target, const int *tokens, const int *parents,
                                  int n_nodes, const float *u, hipStream_t s) {
  if (n_nodes < 0 || n_nodes > DSH_TREE_MAX) return hipErrorInvalidValue;
  const verify_args a{path, result, p, q, u, target, tokens, parents, p_stride, q_stride, vocab, n_nodes};
  k_tree_verify<<<1, VT, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t dsh_launch_tree_commit(const dsh_tree_commit_t *A, hipStream_t s) {
  if (A->n_nodes < 1 || A->n_nodes > DSH_TREE_MAX) return hipErrorInvalidValue;
  const dim3 g(A->acc ? (A->n_cache + A->n_nodes + 255) / 256 : 1, A->cache.n_heads);
#define CASE(D, T)                             \
  case D:                                      \
    k_tree_commit<D, T><<<g, 256, 0, s>>>(*A); \
    break;
  if (A->cache.bf16) {
    BY_DIM(A->cache.head_dim, uint16_t, CASE)
  } else {
    BY_DIM(A->cache.head_dim, float, CASE)
  }
#undef CASE
  return hipGetLastError();
}

}  // extern "C"
