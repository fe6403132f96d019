/* ds_hip_tree.c — drafted tokens over a KV cache: the checks and launches of ds_hip_tree_attention, ds_hip_tree_verify,
 * ds_hip_tree_commit and ds_hip_kv_evict (no counterpart in the reference). */
#include <limits.h>
#include <math.h>
#include <string.h>

#include "ds_hip.h"
#include "dsr.h"

_Static_assert(DS_HIP_TREE_MAX_NODES == DSH_TREE_MAX, "nodes that the kernels hold");

/* The library works on device 0 whatever the caller's thread has made current; leave() puts that back. */
static int enter(int *dev) {
  if (dsr_init()) return -1;
  DSR_TRY(hipGetDevice(dev), "current device");
  if (*dev != 0) DSR_TRY(hipSetDevice(0), "device 0");
  return 0;
}

static int leave(int dev, const char *what, hipError_t e) {
  if (dev != 0) hipSetDevice(dev);
  return e == hipSuccess ? 0 : dsr_fail(what, e);
}

static int aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

/* |x| < 2^62 bytes for everything that is indexed below */
#define STRIDE_MAX ((int64_t)1 << 40)

static int kv_check(const char *what, const char *name, const ds_hip_kv_t *kv, int need) {
  if (!kv) return dsr_failf("%s: %s is NULL", what, name);
  if (kv->dtype != DS_HIP_KV_F32 && kv->dtype != DS_HIP_KV_BF16)
    return dsr_failf("%s: %s: unknown type %d", what, name, kv->dtype);
  const int64_t d = kv->head_dim, unit = kv->dtype == DS_HIP_KV_F32 ? 4 : 8;
  if (d != 64 && d != 128 && d != 192 && d != 256)
    return dsr_failf("%s: %s: head_dim %d (64, 128, 192 or 256)", what, name, kv->head_dim);
  if (kv->n_heads < 1 || kv->n_heads > 1024 || kv->rows < 0)
    return dsr_failf("%s: %s: %d heads, %d rows", what, name, kv->n_heads, kv->rows);
  if (need < 0 || need > kv->rows) return dsr_failf("%s: %s: %d rows of %d", what, name, need, kv->rows);
  if (need == 0) return 0;
  if (!kv->k || !kv->v) return dsr_failf("%s: %s: NULL arrays", what, name);
  if (!aligned16(kv->k) || !aligned16(kv->v) || (kv->rows > 1 && kv->row_stride % unit) ||
      (kv->n_heads > 1 && kv->head_stride % unit))
    return dsr_failf("%s: %s: k, v and the strides must be multiples of 16 bytes", what, name);
  /* rows and heads side by side in one order or the other, none over another */
  const int64_t rs = kv->rows > 1 ? kv->row_stride : d, hs = kv->n_heads > 1 ? kv->head_stride : d;
  if (rs < d || hs < d || rs > STRIDE_MAX || hs > STRIDE_MAX ||
      (rs < (int64_t)(kv->n_heads - 1) * hs + d && hs < (int64_t)(kv->rows - 1) * rs + d))
    return dsr_failf("%s: %s: rows overlap (strides %lld and %lld)", what, name, (long long)rs, (long long)hs);
  return 0;
}

static int kv_same(const ds_hip_kv_t *a, const ds_hip_kv_t *b) {
  return a->n_heads == b->n_heads && a->head_dim == b->head_dim && a->dtype == b->dtype;
}

static dsh_kv_t kv_dev(const ds_hip_kv_t *kv) {
  dsh_kv_t d = {kv->k, kv->v, kv->row_stride, kv->head_stride, kv->n_heads, kv->head_dim, kv->dtype == DS_HIP_KV_BF16};
  return d;
}

/* Whether [a, a + n) and [b, b + m) bytes have one in common. */
static int overlap(const void *a, size_t n, const void *b, size_t m) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + m && y < x + n;
}

int ds_hip_attn_kv_view(const ds_hip_attn_t *A, ds_hip_kv_t *kv) {
  float *k, *v;
  int stride;
  if (!A || !kv) return dsr_failf("ds_hip_attn_kv_view: NULL argument");
  ds_hip_attn_kv(A, &k, &v, &stride);
  kv->k = k;
  kv->v = v;
  kv->row_stride = stride;
  kv->rows = ds_hip_attn_max_seq(A);
  ds_hip_attn_heads(A, &kv->n_heads, &kv->head_dim);
  kv->head_stride = kv->head_dim;
  kv->dtype = DS_HIP_KV_F32;
  return 0;
}

int ds_hip_tree_attention(float *out_dev, int64_t out_stride, float *lse_dev, float *scores_dev, int64_t score_stride,
                          const float *q_dev, int64_t q_stride, int n_heads, const ds_hip_kv_t *cache, int n_cache,
                          const ds_hip_kv_t *tree, const int *parents_dev, int n_nodes, float scale, int prefill_len,
                          int window) {
  static const char *const me = "ds_hip_tree_attention";
  if (!out_dev || !q_dev || !parents_dev) return dsr_failf("%s: NULL argument", me);
  if (n_nodes < 1 || n_nodes > DS_HIP_TREE_MAX_NODES)
    return dsr_failf("%s: %d nodes (1 to %d)", me, n_nodes, DS_HIP_TREE_MAX_NODES);
  if (kv_check(me, "cache", cache, n_cache) || kv_check(me, "tree", tree, n_nodes)) return -1;
  if (!kv_same(cache, tree)) return dsr_failf("%s: cache and tree differ in heads, head_dim or type", me);
  if (n_heads < 1 || n_heads % cache->n_heads || n_heads / cache->n_heads > 1024)
    return dsr_failf("%s: %d query heads over %d", me, n_heads, cache->n_heads);
  if (n_cache > INT_MAX - DS_HIP_TREE_MAX_NODES) return dsr_failf("%s: %d cached rows", me, n_cache);
  const int64_t width = (int64_t)n_heads * cache->head_dim;
  if (q_stride < width || out_stride < width || q_stride % 4 || out_stride % 4 || q_stride > STRIDE_MAX ||
      out_stride > STRIDE_MAX || !aligned16(q_dev) || !aligned16(out_dev))
    return dsr_failf("%s: q and out need rows of %lld floats, strides and addresses multiples of 16 bytes", me,
                     (long long)width);
  if (scores_dev && (score_stride < (int64_t)n_cache + n_nodes || score_stride > STRIDE_MAX))
    return dsr_failf("%s: score_stride %lld is below %d + %d", me, (long long)score_stride, n_cache, n_nodes);
  if (prefill_len < 0 || window < 0 || !isfinite(scale))
    return dsr_failf("%s: prefill_len %d, window %d, scale %g", me, prefill_len, window, (double)scale);
  dsh_tree_attn_t a;
  memset(&a, 0, sizeof a);
  a.cache = kv_dev(cache);
  a.tree = kv_dev(tree);
  a.q = q_dev;
  a.parents = parents_dev;
  a.out = out_dev;
  a.lse = lse_dev;
  a.scores = scores_dev;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.score_stride = score_stride;
  a.n_cache = n_cache;
  a.n_nodes = n_nodes;
  a.n_heads = n_heads;
  a.prefill_len = prefill_len;
  a.window = window;
  a.scale = scale;
  int dev;
  if (enter(&dev)) return -1;
  float *work = (float *)dsr_scratch(DSR_SLOT_TREE, dsh_tree_attention_work(&a) * sizeof(float));
  if (!work) {
    leave(dev, me, hipSuccess);
    return -1;
  }
  return leave(dev, me, dsh_launch_tree_attention(&a, work, dsr_stream));
}

static int verify_check(const char *me, const int *path, const int *result, const int *tokens, const int *parents, int n_nodes) {
  if (n_nodes < 0 || n_nodes > DS_HIP_TREE_MAX_NODES)
    return dsr_failf("%s: %d nodes (0 to %d)", me, n_nodes, DS_HIP_TREE_MAX_NODES);
  if (!result || (n_nodes && (!path || !tokens || !parents))) return dsr_failf("%s: NULL argument", me);
  return 0;
}

/* The words that a verification's blocks tell each other their sums in: zeroed once, every launch with an epoch of its own. */
static unsigned long long *verify_words(void) {
  static void *words = NULL;
  if (words) return (unsigned long long *)words;
  const size_t bytes = (size_t)DSH_VERIFY_WORDS * 8;
  void *p = NULL;
  hipError_t e = hipMalloc(&p, bytes);
  if (e == hipSuccess) e = hipMemsetAsync(p, 0, bytes, dsr_stream);
  if (e != hipSuccess) {
    dsr_fail("verification words", e);
    if (p) hipFree(p);
    return NULL;
  }
  return (unsigned long long *)(words = p);
}

int ds_hip_tree_verify(int *path_dev, int *result_dev, const float *p_dev, int64_t p_stride, const float *q_dev,
                       int64_t q_stride, int vocab, const int *tokens_dev, const int *parents_dev, int n_nodes,
                       const float *u_dev) {
  static const char *const me = "ds_hip_tree_verify";
  if (!p_dev || !u_dev) return dsr_failf("%s: NULL argument", me);
  if (verify_check(me, path_dev, result_dev, tokens_dev, parents_dev, n_nodes)) return -1;
  if (vocab < 1 || vocab > 1 << 30 || (n_nodes > 0 && (p_stride < vocab || (q_dev && q_stride < vocab))) || p_stride > STRIDE_MAX ||
      q_stride > STRIDE_MAX)
    return dsr_failf("%s: vocab %d, strides %lld and %lld", me, vocab, (long long)p_stride, (long long)q_stride);
  int dev;
  if (enter(&dev)) return -1;
  unsigned long long *words = verify_words();
  if (!words) {
    leave(dev, me, hipSuccess);
    return -1;
  }
  return leave(dev, me, dsh_launch_tree_verify(path_dev, result_dev, p_dev, p_stride, q_dev, q_stride, vocab, tokens_dev,
                                               parents_dev, n_nodes, u_dev, words, dsr_expert_epoch(),
                                               dsr_derr_dev(DSR_DERR_VERIFY_WAIT), dsr_stream));
}

int ds_hip_tree_verify_greedy(int *path_dev, int *result_dev, const int *target_dev, const int *tokens_dev,
                              const int *parents_dev, int n_nodes) {
  static const char *const me = "ds_hip_tree_verify_greedy";
  if (!target_dev) return dsr_failf("%s: NULL argument", me);
  if (verify_check(me, path_dev, result_dev, tokens_dev, parents_dev, n_nodes)) return -1;
  int dev;
  if (enter(&dev)) return -1;
  return leave(dev, me, dsh_launch_tree_verify_greedy(path_dev, result_dev, target_dev, tokens_dev, parents_dev, n_nodes,
                                                      dsr_stream));
}

int ds_hip_tree_commit(const ds_hip_kv_t *cache, int n_cache, const ds_hip_kv_t *tree, int n_nodes, const int *path_dev,
                       const int *result_dev, const float *scores_dev, int64_t score_stride, const float *lse_dev,
                       int n_heads, const float *acc_dev, float *acc_out_dev, int64_t acc_stride, int *pos_dev,
                       int64_t pos_stride, int pos0) {
  static const char *const me = "ds_hip_tree_commit";
  if (!path_dev || !result_dev) return dsr_failf("%s: NULL argument", me);
  if (n_nodes < 1 || n_nodes > DS_HIP_TREE_MAX_NODES)
    return dsr_failf("%s: %d nodes (1 to %d)", me, n_nodes, DS_HIP_TREE_MAX_NODES);
  if (n_cache < 0 || n_cache > INT_MAX - DS_HIP_TREE_MAX_NODES) return dsr_failf("%s: %d cached rows", me, n_cache);
  const int n = n_cache + n_nodes;
  if (kv_check(me, "cache", cache, n) || kv_check(me, "tree", tree, n_nodes)) return -1;
  if (!kv_same(cache, tree)) return dsr_failf("%s: cache and tree differ in heads, head_dim or type", me);
  if (!acc_dev != !acc_out_dev) return dsr_failf("%s: acc and acc_out go together", me);
  if (acc_dev) {
    if (!scores_dev || !lse_dev) return dsr_failf("%s: the weights need scores and lse", me);
    if (n_heads < 1 || n_heads % cache->n_heads || n_heads / cache->n_heads > 1024)
      return dsr_failf("%s: %d query heads over %d", me, n_heads, cache->n_heads);
    if (score_stride < n || acc_stride < n || score_stride > STRIDE_MAX || acc_stride > STRIDE_MAX)
      return dsr_failf("%s: strides %lld and %lld are below %d + %d", me, (long long)score_stride, (long long)acc_stride,
                       n_cache, n_nodes);
    const size_t bytes = ((size_t)(cache->n_heads - 1) * acc_stride + n) * 4;
    if (acc_dev != acc_out_dev && overlap(acc_dev, bytes, acc_out_dev, bytes))
      return dsr_failf("%s: acc_out overlaps acc", me);
  }
  if (pos_dev && (pos_stride < n || pos_stride > STRIDE_MAX))
    return dsr_failf("%s: pos_stride %lld is below %d + %d", me, (long long)pos_stride, n_cache, n_nodes);
  if (pos_dev && (pos0 < 0 || pos0 > INT_MAX - DS_HIP_TREE_MAX_NODES)) return dsr_failf("%s: pos0 %d", me, pos0);
  dsh_tree_commit_t a;
  memset(&a, 0, sizeof a);
  a.cache = kv_dev(cache);
  a.tree = kv_dev(tree);
  a.path = path_dev;
  a.result = result_dev;
  a.scores = scores_dev;
  a.lse = lse_dev;
  a.acc = acc_dev;
  a.acc_out = acc_out_dev;
  a.pos = pos_dev;
  a.score_stride = score_stride;
  a.acc_stride = acc_stride;
  a.pos_stride = pos_stride;
  a.n_cache = n_cache;
  a.n_nodes = n_nodes;
  a.n_heads = n_heads;
  a.pos0 = pos0;
  int dev;
  if (enter(&dev)) return -1;
  return leave(dev, me, dsh_launch_tree_commit(&a, dsr_stream));
}

/* An output array [heads][out_stride] of `keep` entries beside its input [heads][stride] of n: the input itself, or apart. */
static int beside(const void *in, int64_t stride, int n, const void *out, int64_t out_stride, int keep, int heads) {
  if (!out || !in) return 1;
  if (in == out) return stride == out_stride || heads == 1;
  return !overlap(in, ((size_t)(heads - 1) * stride + n) * 4, out, ((size_t)(heads - 1) * out_stride + keep) * 4);
}

int ds_hip_kv_evict(const ds_hip_kv_t *cache, int n_rows, int n_keep, const float *acc_dev, int64_t acc_stride,
                    float *acc_out_dev, int64_t acc_out_stride, const int *pos_dev, int64_t pos_stride, int *pos_out_dev,
                    int64_t pos_out_stride, int sink, int recent_from, int *slots_dev) {
  static const char *const me = "ds_hip_kv_evict";
  if (n_rows < 0 || n_rows > 1 << 30 || n_keep < 0 || n_keep > n_rows) return dsr_failf("%s: %d of %d rows", me, n_keep, n_rows);
  if (kv_check(me, "cache", cache, n_rows)) return -1;
  if (!acc_dev) return dsr_failf("%s: NULL argument", me);
  if (pos_out_dev && !pos_dev) return dsr_failf("%s: pos_out without pos", me);
  if (acc_stride < n_rows || (pos_dev && pos_stride < n_rows) || (acc_out_dev && acc_out_stride < n_keep) ||
      (pos_out_dev && pos_out_stride < n_keep) || acc_stride > STRIDE_MAX || pos_stride > STRIDE_MAX ||
      acc_out_stride > STRIDE_MAX || pos_out_stride > STRIDE_MAX)
    return dsr_failf("%s: strides below %d rows (in) or %d (out)", me, n_rows, n_keep);
  if (!beside(acc_dev, acc_stride, n_rows, acc_out_dev, acc_out_stride, n_keep, cache->n_heads) ||
      !beside(pos_dev, pos_stride, n_rows, pos_out_dev, pos_out_stride, n_keep, cache->n_heads))
    return dsr_failf("%s: acc_out and pos_out must be their inputs, with the same stride, or lie apart from them", me);
  if (n_rows == 0 || n_keep == 0) return 0; /* nothing stays, nothing is written */
  dsh_kv_evict_t a;
  memset(&a, 0, sizeof a);
  a.cache = kv_dev(cache);
  a.acc = acc_dev;
  a.pos = pos_dev;
  a.acc_out = acc_out_dev;
  a.pos_out = pos_out_dev;
  a.slots = slots_dev;
  a.acc_stride = acc_stride;
  a.acc_out_stride = acc_out_stride;
  a.pos_stride = pos_stride;
  a.pos_out_stride = pos_out_stride;
  a.n = n_rows;
  a.keep = n_keep;
  a.sink = sink;
  a.recent_from = recent_from;
  int dev;
  if (enter(&dev)) return -1;
  a.work = (int *)dsr_scratch(DSR_SLOT_TREE, dsh_kv_evict_work(cache->n_heads, n_rows, n_keep) * sizeof(int));
  if (!a.work) {
    leave(dev, me, hipSuccess);
    return -1;
  }
  return leave(dev, me, dsh_launch_kv_evict(&a, dsr_stream));
}
