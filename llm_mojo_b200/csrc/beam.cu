// Beam search: the K best of the K x V continuations of each item.
//
// candidate(k, v) = score_k + x_kv - lse_k.  Within a beam the order is that of the logits x, so a first pass needs no log-sum-exp: it reads every
// logit once, a block per (beam, chunk of the vocabulary), and leaves the chunk's maximum, its sum of exponentials and its K best logits, sorted.
// The second pass, one block per item, adds up the log-sum-exp of each beam in 64 bits and merges the sorted lists by their heads.
//
// A column belongs to the same thread and place of the sums whatever the address of its row, so that two beams with the same logits have
// the same log-sum-exp to the last bit and their tie goes to the lower one.
//
// This file has no counterpart in the reference project, which samples (llmm/sampler.mojo:19-66).
#include "common.cuh"
using namespace llmb;

namespace {
constexpr int CHUNK = 4096, THREADS = 256, PER = CHUNK / THREADS, BEAM_MAX = 64;

// a float as an unsigned integer of the same order; -0 and +0 are the same, NaN counts as -inf
__device__ __forceinline__ uint32_t ordered(float x) {
  if (!(x == x)) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x);
  return b >> 63 ? ~b : b | (1ull << 63);
}
// best first: the larger logit, then the lower column
__device__ __forceinline__ unsigned long long key_of(float x, int col) { return (unsigned long long)ordered(x) << 32 | (uint32_t)~col; }

__device__ __forceinline__ unsigned long long warp_max_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o); v = w > v ? w : v; }
  return v;
}

// Workspace: stats [rows][chunks] float2 (maximum, sum of exponentials), lists [rows][chunks][K] of keys.
template <typename T>
__global__ void __launch_bounds__(THREADS) beam_chunk_kernel(float2* __restrict__ stats, unsigned long long* __restrict__ lists, const T* __restrict__ logits,
                                                             const bool* __restrict__ finished, int K, int V, long long ld, int chunks) {
  pdl_trigger();
  pdl_wait();
  __shared__ unsigned long long cand[CHUNK];
  __shared__ float red[THREADS / 32];
  __shared__ uint32_t best_of[THREADS];
  __shared__ int n_cand;
  __shared__ uint32_t threshold;
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if (finished != nullptr && finished[row]) return;    // its one candidate does not depend on its logits
  const int c0 = chunk * CHUNK, w = min(CHUNK, V - c0);
  const T* x = logits + row * ld + c0;
  float v[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) { const int c = j * THREADS + tid; v[j] = c < w ? to_f<T>(x[c]) : -INFINITY; }
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) m = fmaxf(m, v[j]);
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) if (j * THREADS + tid < w) mine = max(mine, ordered(v[j]));
  best_of[tid] = mine;
  m = warp_max(m);
  if (lane == 0) red[warp] = m;
  if (tid == 0) n_cand = 0;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) m = fmaxf(m, red[i]);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) if (j * THREADS + tid < w && !(v[j] == -INFINITY)) s += exp2f((v[j] - m) * 1.4426950408889634f);
  s = warp_sum(s);
  __syncthreads();
  if (lane == 0) red[warp] = s;
  // The K-th largest of the threads' best logits is no larger than the K-th largest of all: what is below it is out.
  if (warp == 0) {
    uint32_t b[THREADS / 32];
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) b[i] = best_of[i * 32 + lane];
    uint32_t t = 0;
    for (int i = 0; i < K; ++i) {
      uint32_t l = 0;
#pragma unroll
      for (int y = 0; y < THREADS / 32; ++y) l = max(l, b[y]);
      t = __reduce_max_sync(0xffffffffu, l);
      const unsigned has = __ballot_sync(0xffffffffu, l == t);
      if (lane == __ffs(has) - 1) {
        bool out = false;
#pragma unroll
        for (int y = 0; y < THREADS / 32; ++y) if (!out && b[y] == t) { b[y] = 0; out = true; }
      }
    }
    if (lane == 0) threshold = t;
  }
  __syncthreads();
  const uint32_t t = threshold;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int c = j * THREADS + tid;
    if (c < w && ordered(v[j]) >= t) cand[atomicAdd(&n_cand, 1)] = key_of(v[j], c0 + c);      // any order: they are sorted below
  }
  __syncthreads();
  if (warp == 0) {
    if (lane == 0) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) sum += red[i];
      stats[(long long)row * chunks + chunk] = make_float2(m, sum);
    }
    const int n = n_cand;
    unsigned long long* out = lists + ((long long)row * chunks + chunk) * K;
    unsigned long long last = ~0ull;
    for (int i = 0; i < K; ++i) {                      // keys differ from one another: the next one is the largest below the last
      unsigned long long b = 0;
      for (int y = lane; y < n; y += 32) { const unsigned long long k = cand[y]; if (k < last && k > b) b = k; }
      last = warp_max_u64(b);
      if (lane == 0) out[i] = last;                    // 0 where the chunk has fewer than K columns
      if (last == 0) { for (int y = i + 1; y < K; ++y) if (lane == 0) out[y] = 0; break; }
    }
  }
}

__global__ void __launch_bounds__(THREADS) beam_merge_kernel(float* __restrict__ scores_out, int* __restrict__ tokens, int* __restrict__ parents,
                                                             bool* __restrict__ finished_out, const float* __restrict__ scores, const bool* __restrict__ finished,
                                                             const float2* __restrict__ stats, const unsigned long long* __restrict__ lists, int K, int V, int eos, int chunks) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ int heads[];                       // [K * chunks] next entry of each list
  __shared__ double lse[BEAM_MAX];
  __shared__ int kind[BEAM_MAX];                       // 0: alive, 1: finished, 2: offers nothing
  __shared__ float out_score[BEAM_MAX];
  const int item = blockIdx.x, tid = threadIdx.x, lane = tid % 32;
  for (int k = tid / 32; k < K; k += THREADS / 32) {
    const long long row = (long long)item * K + k;
    const float sc = scores[row];
    const bool fin = finished != nullptr && finished[row], ok = fabsf(sc) <= 3.402823466e38f;
    float m = -INFINITY;
    double sum = 0.0;
    if (!fin) {
      for (int c = lane; c < chunks; c += 32) m = fmaxf(m, stats[row * chunks + c].x);
      m = warp_max(m);
      for (int c = lane; c < chunks; c += 32) {
        const float2 s = stats[row * chunks + c];
        if (!(s.x == -INFINITY && s.y == 0.f)) sum += (double)s.y * exp((double)s.x - (double)m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane == 0) {
      const double l = (double)m + log(sum);
      lse[k] = l;
      kind[k] = !ok ? 2 : fin ? 1 : l - l == 0.0 ? 0 : 2;
    }
  }
  for (int i = tid; i < K * chunks; i += THREADS) heads[i] = 0;
  __syncthreads();
  if (tid >= 32) return;
  // The lists' heads, one after another; a beam that is not alive has one list of its own making in the place of its first chunk's.
  for (int i = 0; i < K; ++i) {
    unsigned long long bk = 0;                         // of the best head: its ordered value, its flat index, its list
    uint32_t bi = 0xffffffffu;
    int bl = -1;
    for (int l = lane; l < K * chunks; l += 32) {
      const int k = l / chunks, h = heads[l], kd = kind[k];
      const long long row = (long long)item * K + k;
      double val = -INFINITY;
      int col;
      if (h >= K) continue;
      if (kd == 0) {
        const unsigned long long e = lists[(row * chunks + l % chunks) * K + h];
        if (e == 0) continue;
        col = (int)~(uint32_t)e;
        val = (double)scores[row] + ((double)unordered((uint32_t)(e >> 32)) - lse[k]);
      } else {
        if (l % chunks != 0) continue;
        if (kd == 1) {                                 // eos first, then the others, which are all at -inf
          col = h == 0 ? eos : h - 1 < eos ? h - 1 : h;
          if (h == 0) val = (double)scores[row];
        } else col = h;
      }
      const unsigned long long key = ordered(val + 0.0);
      const uint32_t idx = (uint32_t)k * (uint32_t)V + (uint32_t)col;
      if (key > bk || (key == bk && idx < bi)) { bk = key; bi = idx; bl = l; }
    }
    const unsigned long long top = warp_max_u64(bk);
    const uint32_t idx = __reduce_min_sync(0xffffffffu, bk == top ? bi : 0xffffffffu);
    if (bl >= 0 && bk == top && bi == idx) {           // one lane: flat indexes differ
      heads[bl] += 1;
      const int k = (int)(idx / (uint32_t)V), tok = (int)(idx % (uint32_t)V);
      const unsigned long long b = top >> 63 ? top ^ (1ull << 63) : ~top;
      const long long at = (long long)item * K + i;
      out_score[i] = (float)__longlong_as_double((long long)b);
      scores_out[at] = out_score[i];
      tokens[at] = tok;
      parents[at] = k;
      if (finished_out != nullptr) finished_out[at] = tok == eos || kind[k] == 1 || (finished != nullptr && finished[(long long)item * K + k]);
    }
    __syncwarp();
  }
}
}  // namespace

// The arguments of a call as the Python side (ops/beam.py) packs them.  work: B K chunks (8 + 8 K) bytes.
struct BeamSelectArgs {
  float* scores_out; int *tokens, *parents; bool* finished_out;          // finished_out: optional
  const void* logits; const float* scores; const bool* finished;         // finished: optional
  void* work;
  long long ld;
  int B, K, V, eos, dtype, pad;
};

LLMB_API int llmb_beam_select(const BeamSelectArgs* a, cudaStream_t st) {
  const int K = a->K, V = a->V, chunks = ceil_div(V, CHUNK), rows = a->B * K;
  if (K < 1 || K > BEAM_MAX || rows > 65535 || (long long)K * chunks * 4 > 40 * 1024) return LLMB_ERR_BAD_ARG;
  float2* stats = (float2*)a->work;
  unsigned long long* lists = (unsigned long long*)(stats + (long long)rows * chunks);
  const dim3 grid(chunks, rows);
  int rc = a->dtype == LLMB_BF16
               ? launch_pdl(beam_chunk_kernel<__nv_bfloat16>, grid, THREADS, 0, st, stats, lists, (const __nv_bfloat16*)a->logits, a->finished, K, V, a->ld, chunks)
               : launch_pdl(beam_chunk_kernel<float>, grid, THREADS, 0, st, stats, lists, (const float*)a->logits, a->finished, K, V, a->ld, chunks);
  if (rc) return rc;
  return launch_pdl(beam_merge_kernel, a->B, THREADS, (size_t)K * chunks * 4, st, a->scores_out, a->tokens, a->parents, a->finished_out, a->scores, a->finished,
                    (const float2*)stats, (const unsigned long long*)lists, K, V, a->eos, chunks);
}
