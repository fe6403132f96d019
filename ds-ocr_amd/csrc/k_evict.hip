// k_evict.hip — which rows of a KV cache stay (k_kv_evict: per head the rows with the least attention weight go), and the
// moves that bring them together.
#include "dsh.h"
#include "k_core.h"

#define ET 1024

// Floats in ascending order as unsigned numbers; -0 as 0, a NaN as -inf.
__device__ __forceinline__ uint32_t evict_key(float a) {
  if (a != a) a = -__builtin_huge_valf();
  const uint32_t u = __float_as_uint(a + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum of v over the block's threads; *total receives the sum.
__device__ int evict_scan(int v, int *s_w, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int a = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int b = __shfl_up(a, o);
    if (lane >= o) a += b;
  }
  __syncthreads();
  if (lane == 63) s_w[wave] = a;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < ET / 64; w++) {
    before += w < wave ? s_w[w] : 0;
    all += s_w[w];
  }
  *total = all;
  return before + a - v;
}

// One block per head: the threshold by radix select over 8-bit digits, then the rows that go, the holes they leave below
// `keep` and the rows that fill them.
template <int D, typename T>
__global__ void __launch_bounds__(ET) k_kv_evict(dsh_kv_evict_t A) {
  __shared__ int s_hist[256], s_w[ET / 64], s_digit, s_left;
  const int h = blockIdx.x, n = A.n, keep = A.keep, tid = threadIdx.x;
  const float *acc = A.acc + h * A.acc_stride;
  const int *pos = A.pos ? A.pos + h * A.pos_stride : nullptr;
  auto guarded = [&](int j) {
    const int p = pos ? pos[j] : j;
    return p < A.sink || p >= A.recent_from;
  };
  int v = 0, total;
  for (int j = tid; j < n; j += ET) v += !guarded(j);
  evict_scan(v, s_w, &total);
  int gone = n - keep;               // rows that go
  const bool all_free = gone > total;  // every unguarded row, and some of the guarded
  if (all_free) gone -= total;
  // among the rows of the class (guarded == all_free) the `gone` lowest go: the gone-th key, digit by digit
  uint32_t prefix = 0;
  int left = gone;  // how many of those with the prefix so far
  for (int shift = 24; shift >= 0 && gone > 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += ET) {
      const uint32_t k = evict_key(acc[j]);
      if (guarded(j) == all_free && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))))
        atomicAdd(&s_hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    int all;
    const int c = tid < 256 ? s_hist[tid] : 0;
    const int before = evict_scan(c, s_w, &all);
    if (before < left && before + c >= left) {
      s_digit = tid;
      s_left = left - before;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    left = s_left;
  }
  // a thread's rows are consecutive: ranks in the order of the rows by one scan
  const int per = (n + ET - 1) / ET, j0 = min(tid * per, n), j1 = min(j0 + per, n);
  int ties = 0;
  for (int j = j0; j < j1; j++) ties += gone > 0 && guarded(j) == all_free && evict_key(acc[j]) == prefix;
  const int tie0 = evict_scan(ties, s_w, &total);
  auto stays = [&](int j, int &tie) {
    const bool g = guarded(j);
    if (g != all_free) return g;  // guarded rows stay; unguarded ones go when the class is the guarded
    if (gone == 0) return true;
    const uint32_t k = evict_key(acc[j]);
    if (k != prefix) return k > prefix;
    return tie++ >= left;
  };
  int holes = 0, movers = 0, tie = tie0;
  for (int j = j0; j < j1; j++) {
    const bool s = stays(j, tie);
    holes += j < keep && !s;
    movers += j >= keep && s;
  }
  int *mv = A.work + (int64_t)h * (n - keep), *slot = A.work + (int64_t)A.cache.n_heads * (n - keep) + (int64_t)h * keep;
  int hole = evict_scan(holes, s_w, &total), mover = evict_scan(movers, s_w, &total);
  tie = tie0;
  for (int j = j0; j < j1; j++)
    if (stays(j, tie) && j >= keep) mv[mover++] = j;
  __syncthreads();
  tie = tie0;
  for (int j = j0; j < min(j1, keep); j++) slot[j] = stays(j, tie) ? j : mv[hole++];
  __syncthreads();
  float a = 0.0f;
  for (int j = tid; j < keep; j += ET) {
    const int from = slot[j];
    if (A.slots) A.slots[(int64_t)h * keep + j] = from;
    if (A.acc_out) {
      a = acc[from];
      A.acc_out[h * A.acc_out_stride + j] = a;
    }
    if (A.pos_out) A.pos_out[h * A.pos_out_stride + j] = pos[from];
  }
  for (int j = tid >> 6; j < keep; j += ET / 64) {
    const int from = slot[j];
    if (from == j) continue;
    const int64_t x = from * A.cache.row_stride + h * A.cache.head_stride, y = j * A.cache.row_stride + h * A.cache.head_stride;
    for (int d = tid & 63; d < D; d += 64) {
      ((T *)A.cache.k)[y + d] = ((const T *)A.cache.k)[x + d];
      ((T *)A.cache.v)[y + d] = ((const T *)A.cache.v)[x + d];
    }
  }
}

extern "C" {

// Per head the rows that move (n - keep at most) and the row of each slot.
size_t dsh_kv_evict_work(int n_heads, int n, int keep) { return (size_t)n_heads * n; }

hipError_t dsh_launch_kv_evict(const dsh_kv_evict_t *A, hipStream_t s) {
#define EV(D)                                                          \
  case D:                                                              \
    if (A->cache.bf16)                                                 \
      k_kv_evict<D, uint16_t><<<A->cache.n_heads, ET, 0, s>>>(*A);     \
    else                                                               \
      k_kv_evict<D, float><<<A->cache.n_heads, ET, 0, s>>>(*A);        \
    break;
  switch (A->cache.head_dim) {
    EV(64) EV(128) EV(192) EV(256)
    default:
      return hipErrorInvalidValue;
  }
#undef EV
  return hipGetLastError();
}

}  // extern "C"
