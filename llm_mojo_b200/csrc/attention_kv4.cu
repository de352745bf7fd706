// Attention of new tokens over the 4-bit key/value cache (layout: kv4.cuh).
//
// A row is one (new token, query head); the rows of a key head share its keys.  o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m) with
// s_j = q k_j scale log2(e) over the positions j that the row's token sees.
//
// This file has no counterpart in the reference project, whose inference keeps no cache (infer_gpt2.mojo:56-144).
#include "kv4.cuh"
#include <cooperative_groups.h>
using namespace llmb;
using namespace kv4;
namespace cg = cooperative_groups;

namespace {
struct Kv4Attn {
  Kv4Desc d;
  void* out; const void* q;
  const int *lens, *counts, *pages;
  int layer, n, group, splits;
  float scale_log2;
  long long qb, qt, qh, ob, ot, oh;                    // element strides
  int* status;
};

// The simple form, in fp32 arithmetic on the FMA pipe.  A cluster of `splits` blocks of eight warps takes R rows of one (slot, key head); the warps
// take chunks of 32 keys in turns.  Scores: one key per lane; values: every lane keeps its own two or four columns.  The warps' and the
// blocks' partial results are joined through (distributed) shared memory.
constexpr int FW = 8;
template <typename T, int HD, int R>
__global__ void __launch_bounds__(FW * 32) attention_kv4_fma_kernel(const Kv4Attn p) {
  constexpr int NB = HD / BLOCK, VB = HD <= 64 ? 1 : 2, LANES = HD / 2 / VB;
  __shared__ float sq[R][HD], pm[FW][R], pl[FW][R], po[FW][R][HD];
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits, h = blockIdx.y, s = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int len = min(max(p.lens[s], 0), p.d.capacity), cnt = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
  const int r0 = tile * R, rows = min(R, cnt * p.group - r0);
  if (rows <= 0) return;                               // the same in every block of the cluster
  int see[R];                                          // keys that row r sees
#pragma unroll
  for (int r = 0; r < R; ++r) see[r] = r < rows ? max(0, min(len, len - cnt + (r0 + r) / p.group + 1)) : 0;
  int most = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) most = max(most, see[r]);
  for (int x = threadIdx.x; x < R * HD; x += FW * 32) {
    const int r = x / HD, i = (r0 + r) / p.group, g = (r0 + r) % p.group;
    sq[r][x % HD] = r < rows ? to_f<T>(reinterpret_cast<const T*>(p.q)[s * p.qb + i * p.qt + (h * p.group + g) * p.qh + x % HD]) * p.scale_log2 : 0.f;
  }
  __syncthreads();
  const long long code0 = p.layer * p.d.code_layer + (long long)h * p.d.capacity * (HD / 2);
  const long long scale0 = p.layer * p.d.scale_layer + (long long)h * p.d.capacity * NB;
  const float kunit = pow2(p.d.k_exp), vunit = pow2(p.d.v_exp);
  float m[R], l[R], acc[R][2 * VB];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < 2 * VB; ++c) acc[r][c] = 0.f;
  }
  for (int base = (split * FW + warp) * 32; base < most; base += p.splits * FW * 32) {
    int slot = s;
    if (p.pages) slot = p.pages[(long long)s * (p.d.capacity / PAGE) + base / PAGE];
    const bool wrong = slot < 0 || slot >= p.d.slots;
    if (wrong) slot = s;
    const int key = base + lane;
    const long long crow = code0 + slot * p.d.code_slot, frow = scale0 + slot * p.d.scale_slot;
    float sc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) sc[r] = 0.f;
    if (key < most) {
      const uint8_t* kc = p.d.kc + crow + (long long)key * (HD / 2);
      const uint8_t* kf = p.d.ks + frow + (long long)key * NB;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint2 w = *reinterpret_cast<const uint2*>(kc + b * 8);
        const float f = wrong ? __int_as_float(0x7fc00000) : e4m3_f32(kf[b]) * kunit;
        float part[R];
#pragma unroll
        for (int r = 0; r < R; ++r) part[r] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 v = f16x2_f32(e2m1x2_f16x2(((j < 4 ? w.x : w.y) >> (8 * (j & 3))) & 0xff));
#pragma unroll
          for (int r = 0; r < R; ++r) part[r] += v.x * sq[r][b * 16 + 2 * j] + v.y * sq[r][b * 16 + 2 * j + 1];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) sc[r] += part[r] * f;
      }
    }
    float pr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (key >= see[r]) sc[r] = -INFINITY;
      const float mn = fmaxf(m[r], warp_max(sc[r])), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m[r] - ref);
      pr[r] = exp2f(sc[r] - ref);
      l[r] = l[r] * alpha + pr[r];
      m[r] = mn;
#pragma unroll
      for (int c = 0; c < 2 * VB; ++c) acc[r][c] *= alpha;
    }
    const int keys = min(32, most - base);
    const uint8_t* vc = p.d.vc + crow + (long long)base * (HD / 2) + lane * VB;
    const uint8_t* vf = p.d.vs + frow + (long long)base * NB + lane * VB * 2 / BLOCK;
    for (int k = 0; k < keys; ++k) {
      float v[2 * VB];
#pragma unroll
      for (int c = 0; c < 2 * VB; ++c) v[c] = 0.f;
      if (lane < LANES) {
        // a NaN scale becomes a number here: the key's scales are NaN as well, and say so to the rows that see it and to no other
        const float f = fminf(e4m3_f32(vf[(long long)k * NB]), 448.f) * vunit;
#pragma unroll
        for (int c = 0; c < VB; ++c) {
          const float2 t = f16x2_f32(e2m1x2_f16x2(vc[(long long)k * (HD / 2) + c]));
          v[2 * c] = t.x * f; v[2 * c + 1] = t.y * f;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float w = __shfl_sync(0xffffffffu, pr[r], k);
#pragma unroll
        for (int c = 0; c < 2 * VB; ++c) acc[r][c] += w * v[c];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float t = warp_sum(l[r]);
    if (lane == 0) { pm[warp][r] = m[r]; pl[warp][r] = t; }
    if (lane < LANES) {
#pragma unroll
      for (int c = 0; c < 2 * VB; ++c) po[warp][r][lane * VB * 2 + c] = acc[r][c];
    }
  }
  __syncthreads();
  // the block's warps into part 0, then the cluster's blocks, each of which finishes a share of the elements
  for (int x = threadIdx.x; x < R * HD; x += FW * 32) {
    const int r = x / HD, c = x % HD;
    float mx = pm[0][r], o = 0.f;
#pragma unroll
    for (int w = 1; w < FW; ++w) mx = fmaxf(mx, pm[w][r]);
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < FW; ++w) o += po[w][r][c] * exp2f(pm[w][r] - ref);
    po[0][r][c] = o;
  }
  __syncthreads();
  if (threadIdx.x < R) {
    const int r = threadIdx.x;
    float mx = pm[0][r], t = 0.f;
#pragma unroll
    for (int w = 1; w < FW; ++w) mx = fmaxf(mx, pm[w][r]);
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < FW; ++w) t += pl[w][r] * exp2f(pm[w][r] - ref);
    pm[0][r] = mx; pl[0][r] = t;
  }
  if (p.splits > 1) cluster.sync(); else __syncthreads();
  for (int x = split * (FW * 32) + threadIdx.x; x < rows * HD; x += p.splits * FW * 32) {
    const int r = x / HD, c = x % HD;
    float mx = -INFINITY, o = 0.f, t = 0.f;
    for (int k = 0; k < p.splits; ++k) mx = fmaxf(mx, *cluster.map_shared_rank(&pm[0][r], k));
    const float ref = mx == -INFINITY ? 0.f : mx;
    for (int k = 0; k < p.splits; ++k) {
      const float w = exp2f(*cluster.map_shared_rank(&pm[0][r], k) - ref);
      t += *cluster.map_shared_rank(&pl[0][r], k) * w;
      o += *cluster.map_shared_rank(&po[0][r][c], k) * w;
    }
    const int i = (r0 + r) / p.group, g = (r0 + r) % p.group;
    reinterpret_cast<T*>(p.out)[s * p.ob + i * p.ot + (h * p.group + g) * p.oh + c] = from_f<T>(t == 0.f ? 0.f : o / t);
  }
  if (p.splits > 1) cluster.sync();                    // no block leaves while another reads its shared memory
}

template <typename T, int HD, int R>
int run_fma(Kv4Attn p, cudaStream_t st) {
  const long long tiles = ceil_div_ll((long long)p.n * p.group, R), ctas = tiles * p.d.heads * p.d.slots;
  p.splits = 1;
  while (p.splits < 8 && ctas * p.splits < 2 * sm_count() && p.splits * FW * 32 < p.d.capacity) p.splits *= 2;
  return launch_pdl_cluster(dim3(p.splits), attention_kv4_fma_kernel<T, HD, R>, dim3((unsigned)(tiles * p.splits), p.d.heads, p.d.slots), FW * 32, 0, st, p);
}
template <typename T, int HD>
int run(const Kv4Attn& p, cudaStream_t st) {
  return (long long)p.n * p.group == 1 ? run_fma<T, HD, 1>(p, st) : run_fma<T, HD, 4>(p, st);
}
template <typename T>
int run_type(const Kv4Attn& p, cudaStream_t st) {
  switch (p.d.head_size) {
    case 32: return run<T, 32>(p, st);
    case 64: return run<T, 64>(p, st);
    case 80: return run<T, 80>(p, st);
    case 96: return run<T, 96>(p, st);
    case 128: return run<T, 128>(p, st);
    default: return LLMB_ERR_BAD_ARG;
  }
}
}  // namespace

LLMB_API int llmb_attention_kv4(const Kv4Desc* d, int layer, void* out, const void* q, const int* lens, const int* counts, const int* pages, int n, int heads,
                                float scale, long long qb, long long qt, long long qh, long long ob, long long ot, long long oh, int dtype, int* status,
                                cudaStream_t st) {
  if (heads % d->heads || d->heads > 65535 || d->slots > 65535) return LLMB_ERR_BAD_ARG;
  Kv4Attn p{*d, out, q, lens, counts, pages, layer, n, heads / d->heads, 1, scale * 1.4426950408889634f, qb, qt, qh, ob, ot, oh, status};
  return dtype == LLMB_BF16 ? run_type<__nv_bfloat16>(p, st) : run_type<float>(p, st);
}
