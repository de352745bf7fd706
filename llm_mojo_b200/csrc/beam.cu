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
constexpr int THREADS = 256, BEAM_MAX = 64;            // a chunk: PER columns for each of THREADS threads, PER 16 or 32

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

// the largest of a warp's keys, to all lanes: the upper halves first, then the lower ones of those that have it
__device__ __forceinline__ unsigned long long warp_max_u64(unsigned long long v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// Workspace: stats [rows][chunks] float2 (maximum, sum of exponentials), lists [rows][chunks][K] of keys.
//
// Each warp takes the j-th best of its lanes' best, j = K / 8 rounded up; no fewer than K logits are not below the least of the eight.  What is
// not below it (some thirty of 4096 for K = 8) is ranked by counting.  Where more than CAND stay (ties) the list is taken from the registers one by one.
// The largest of the warps' K-th best, the threshold before, took K rounds and left over a hundred for K = 16: 16 x 16 beams 41 us, now
// (merge included, see there) 27.
constexpr int CAND = 512, RANKED = THREADS;
template <typename T, int PER>
__global__ void __launch_bounds__(THREADS, PER == 32 ? 4 : 6) beam_chunk_kernel(float2* __restrict__ stats, unsigned long long* __restrict__ lists, const T* __restrict__ logits,
                                                             const bool* __restrict__ finished, int K, int V, long long ld, int chunks) {
  pdl_trigger();
  pdl_wait();
  constexpr int WARPS = THREADS / 32, CHUNK = PER * THREADS;
  __shared__ unsigned long long cand[CAND], best_of[WARPS];
  __shared__ float red[WARPS];
  __shared__ uint32_t level[WARPS];
  __shared__ int n_cand;
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if (finished != nullptr && finished[row]) return;    // its one candidate does not depend on its logits
  const int c0 = chunk * CHUNK, w = min(CHUNK, V - c0);
  const T* x = logits + row * ld + c0;
  float v[PER];
  if (w == CHUNK) {
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = to_f<T>(x[j * THREADS + tid]);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) { const int c = j * THREADS + tid; v[j] = c < w ? to_f<T>(x[c]) : -INFINITY; }
  }
  if (tid == 0) n_cand = 0;
  float m = v[0];
  uint32_t mine = 0;
#pragma unroll
  for (int j = 1; j < PER; ++j) m = fmaxf(m, v[j]);
  if (tid < w) mine = ordered(m);                      // a thread has columns if it has the first
  const float wm = warp_max(m);
  if (lane == 0) red[warp] = wm;
  uint32_t t = 0;
  for (int i = 0; i < K; i += WARPS) {
    t = __reduce_max_sync(0xffffffffu, mine);
    if (lane == __ffs(__ballot_sync(0xffffffffu, mine == t)) - 1) mine = 0;
  }
  if (lane == 0) level[warp] = t;
  __syncthreads();
  m = red[0]; t = level[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) { m = fmaxf(m, red[i]); t = min(t, level[i]); }
  const float safe = m == -INFINITY ? 0.f : m, level_f = unordered(t);
  float2 s2 = make_float2(0.f, 0.f);
  const float2 minus = make_float2(-safe, -safe), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
  unsigned above = 0;                                  // bit per element that stays; a NaN may go, its beam offers nothing
#pragma unroll
  for (int j = 0; j < PER; j += 2) {
    const float2 e = __fmul2_rn(__fadd2_rn(make_float2(v[j], v[j + 1]), minus), log2e);
    s2 = __fadd2_rn(s2, make_float2(ex2(e.x), ex2(e.y)));
    if (v[j] >= level_f) above |= 1u << j;
    if (v[j + 1] >= level_f) above |= 2u << j;
  }
  float s = s2.x + s2.y;
  if (t == 0) above = 0xffffffffu;                     // a warp with fewer lanes in use
  if (w != CHUNK) above &= tid < w ? (2u << (w - 1 - tid) / THREADS) - 1 : 0u;      // columns that there are
  s = warp_sum(s);
  const unsigned kept = above;
  if (above) {
    int at = atomicAdd(&n_cand, __popc(above));        // any order: they are ranked below
    while (above) {                                    // mostly one, read again
      const int c = (__ffs(above) - 1) * THREADS + tid;
      above &= above - 1;
      if (at < CAND) cand[at] = key_of(to_f<T>(x[c]), c0 + c);
      ++at;
    }
  }
  __syncthreads();
  if (lane == 0) red[warp] = s;
  const int n = n_cand;
  unsigned long long* out = lists + ((long long)row * chunks + chunk) * K;
  if (n <= RANKED) {
    if (tid < n) {
      const unsigned long long k = cand[tid];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += cand[i] > k;                   // keys differ from one another
      if (rank < K) out[rank] = k;
    }
    if (n + tid < K) out[n + tid] = 0;                 // fewer columns than K
  } else {
    unsigned long long last = ~0ull;
    for (int i = 0; i < K; ++i) {                      // the largest key below the last
      unsigned long long b = 0;
      if (n <= CAND) {
        for (int y = tid; y < n; y += THREADS) { const unsigned long long k = cand[y]; if (k < last && k > b) b = k; }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (kept >> j & 1) { const unsigned long long k = key_of(v[j], c0 + j * THREADS + tid); if (k < last && k > b) b = k; }
      }
      b = warp_max_u64(b);
      if (lane == 0) best_of[warp] = b;
      __syncthreads();
      last = best_of[0];
#pragma unroll
      for (int y = 1; y < WARPS; ++y) last = best_of[y] > last ? best_of[y] : last;
      if (tid == 0) out[i] = last;                     // 0 where the chunk has fewer than K columns; nothing is below 0
      __syncthreads();
    }
  }
  __syncthreads();
  if (tid == 0) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) sum += red[i];
    stats[(long long)row * chunks + chunk] = make_float2(m, sum);
  }
}

// One block per item.  Its warps add up the log-sum-exps; then one warp merges the sorted lists by their heads, whose values it keeps in shared
// memory; the lists come along where they fit (`staged`).  A beam that is not alive has one list of its own making in the place of its
// first chunk's.
__global__ void __launch_bounds__(THREADS) beam_merge_kernel(float* __restrict__ scores_out, int* __restrict__ tokens, int* __restrict__ parents,
                                                             bool* __restrict__ finished_out, const float* __restrict__ scores, const bool* __restrict__ finished,
                                                             const float2* __restrict__ stats, const unsigned long long* __restrict__ lists, int K, int V, int eos, int chunks,
                                                             int staged) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ unsigned long long sm[];
  __shared__ double lse[BEAM_MAX];
  __shared__ float score[BEAM_MAX];
  __shared__ int kind[BEAM_MAX];                       // 0: alive, 1: finished, 2: offers nothing
  __shared__ bool fin[BEAM_MAX];
  __shared__ unsigned long long won[BEAM_MAX];
  __shared__ uint32_t won_flat[BEAM_MAX];
  const int item = blockIdx.x, tid = threadIdx.x, lane = tid % 32, n_lists = K * chunks;
  unsigned long long* const value = sm;                // [n_lists] ordered value of each list's head, 0: none left
  uint32_t* const flat = reinterpret_cast<uint32_t*>(sm + n_lists);      // its k V + v
  int* const next = reinterpret_cast<int*>(flat + n_lists);              // its beam, and the entry behind it
  unsigned long long* const stage = sm + 2 * n_lists;
  const unsigned long long* mine = lists + (long long)item * n_lists * K;
  if (staged)                                          // all in flight at once, while the log-sum-exps are made
    for (int i = tid; i < n_lists * K; i += THREADS)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((uint32_t)__cvta_generic_to_shared(&stage[i])), "l"(mine + i) : "memory");
  for (int k = tid / 32; k < K; k += THREADS / 32) {
    const long long row = (long long)item * K + k;
    const float sc = scores[row];
    const bool f = finished != nullptr && finished[row], ok = fabsf(sc) <= 3.402823466e38f;
    float m = -INFINITY;
    double sum = 0.0;
    if (!f) {
      for (int c = lane; c < chunks; c += 32) m = fmaxf(m, stats[row * chunks + c].x);
      m = warp_max(m);
      for (int c = lane; c < chunks; c += 32) {
        const float2 s = stats[row * chunks + c];
        if (!(s.x == -INFINITY && s.y == 0.f)) sum += (double)s.y * (double)ex2((s.x - m) * 1.4426950408889634f);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane == 0) {
      const double l = (double)m + log(sum);
      lse[k] = l; score[k] = sc; fin[k] = f;
      kind[k] = !ok ? 2 : f ? 1 : l - l == 0.0 ? 0 : 2;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // entry e of list l, one of beam k's, becomes its head
  auto advance = [&](int l, int k, int e) {
    const int kd = kind[k];
    unsigned long long val = 0;
    int col = 0;
    if (e < K) {
      if (kd == 0) {
        const unsigned long long x = staged ? stage[l * K + e] : mine[(long long)l * K + e];
        if (x != 0) { col = (int)~(uint32_t)x; val = ordered((double)score[k] + ((double)unordered((uint32_t)(x >> 32)) - lse[k]) + 0.0); }
      } else if (l == k * chunks) {                    // finished: eos first; then, or if it offers nothing, the others, all at -inf
        col = kd == 2 ? e : e == 0 ? eos : e - 1 < eos ? e - 1 : e;
        val = ordered(kd == 1 && e == 0 ? (double)score[k] + 0.0 : (double)-INFINITY);
      }
    }
    value[l] = val; flat[l] = (uint32_t)k * (uint32_t)V + (uint32_t)col; next[l] = k << 8 | (e + 1);
  };
  for (int l = tid; l < n_lists; l += THREADS) advance(l, l / chunks, 0);
  __syncthreads();
  if (tid >= 32) return;
  // Every lane keeps the best head of its lists; the one that has the best of all takes the next of that list.  Rounds wait for one another: what can
  // be is done behind them.
  unsigned long long bk;
  uint32_t bi;
  int bl;
  auto look = [&]() {
    bk = 0; bi = 0xffffffffu; bl = -1;
#pragma unroll 8
    for (int l = lane; l < n_lists; l += 32) {
      const unsigned long long x = value[l];
      if (x > bk || (x == bk && x != 0 && flat[l] < bi)) { bk = x; bi = flat[l]; bl = l; }
    }
  };
  look();
  for (int i = 0; i < K; ++i) {
    const unsigned long long top = warp_max_u64(bk);
    const uint32_t idx = __reduce_min_sync(0xffffffffu, bk == top ? bi : 0xffffffffu);
    if (bl >= 0 && bk == top && bi == idx) {           // one lane: flat indexes differ
      won[i] = top; won_flat[i] = idx;
      const int n = next[bl];
      advance(bl, n >> 8, n & 255);
      look();
    }
    __syncwarp();
  }
  for (int i = lane; i < K; i += 32) {
    const unsigned long long x = won[i];
    const int k = (int)(won_flat[i] / (uint32_t)V), tok = (int)(won_flat[i] - (uint32_t)k * (uint32_t)V);
    const long long at = (long long)item * K + i;
    scores_out[at] = (float)__longlong_as_double((long long)(x >> 63 ? x ^ (1ull << 63) : ~x));
    tokens[at] = tok;
    parents[at] = k;
    if (finished_out != nullptr) finished_out[at] = tok == eos || fin[k];
  }
}
}  // namespace

// The arguments of a call as the Python side (ops/beam.py) packs them; the workspace is B K (8 + 8 K) bytes for each 8192 columns.
struct BeamSelectArgs {
  float* scores_out; int *tokens, *parents; bool* finished_out;          // finished_out: optional
  const void* logits; const float* scores; const bool* finished;         // finished: optional
  long long ld;
  int B, K, V, eos, dtype, pad;
};

LLMB_API int llmb_beam_select(const BeamSelectArgs* a, void* work, cudaStream_t st) {
  const int K = a->K, V = a->V, rows = a->B * K;
  // Chunks of 8192 columns, 4096 where that is all there are: fewer blocks with fewer lists to merge, although a chip that they do not fill waits for each
  // of them longer (48 x 8 beams over 50257 columns, fp32: 27.7 us in chunks of 4096, 24.1 of 8192, 32.3 with the registers that leave two blocks on an SM
  // instead of four; 1 x 4 in bf16 7.2 and 7.2, 7 x 8 14.2 and 11.3; 43 x 3 over 2044 columns 7.0 and 7.5).
  const bool wide = V > 4096;
  const int chunks = ceil_div(V, 8192);
  if (K < 1 || K > BEAM_MAX || rows > 65535 || (long long)K * chunks * 16 > 46 * 1024) return LLMB_ERR_BAD_ARG;
  float2* stats = (float2*)work;
  unsigned long long* lists = (unsigned long long*)(stats + (long long)rows * chunks);
  const dim3 grid(chunks, rows);
  auto chunk = [&](auto kernel, auto* logits) { return launch_pdl(kernel, grid, THREADS, 0, st, stats, lists, logits, a->finished, K, V, a->ld, chunks); };
  const __nv_bfloat16* lb = (const __nv_bfloat16*)a->logits;
  const float* lf = (const float*)a->logits;
  int rc;
  if (a->dtype == LLMB_BF16) rc = wide ? chunk(beam_chunk_kernel<__nv_bfloat16, 32>, lb) : chunk(beam_chunk_kernel<__nv_bfloat16, 16>, lb);
  else rc = wide ? chunk(beam_chunk_kernel<float, 32>, lf) : chunk(beam_chunk_kernel<float, 16>, lf);
  if (rc) return rc;
  const size_t heads = (size_t)K * chunks * 16, staged = (size_t)K * chunks * K * 8;
  const bool stage = heads + staged <= 48 * 1024 - 2048;                 // what a block may have without asking
  return launch_pdl(beam_merge_kernel, a->B, THREADS, stage ? heads + staged : heads, st, a->scores_out, a->tokens, a->parents, a->finished_out, a->scores, a->finished,
                    (const float2*)stats, (const unsigned long long*)lists, K, V, a->eos, chunks, (int)stage);
}
