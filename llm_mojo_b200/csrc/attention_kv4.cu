// Attention of new tokens over the 4-bit key/value cache (layout: kv4.cuh).
//
// A row is one (new token, query head); the rows of a key head share its keys.  o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m) with
// s_j = q k_j scale log2(e) over the positions j that the row's token sees.
//
// This file has no counterpart in the reference project, whose inference keeps no cache (infer_gpt2.mojo:56-144).
#include "kv4.cuh"
#include "tc05.cuh"
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

// The form on the tensor core, for bf16 and fp32.  The products are taken transposed, S^T = K q^T and o^T = V^T P^T (mma.sync m16n8k16, f16
// operands, fp32 sums): 16 keys fill a tile's rows and eight columns are rows of q, so that a single query pads to 8 and not to 128
// (as it would in a tcgen05 product), and the codes go from shared memory to registers straight into operands:
//   K  a lane holds contiguous words of a key's row; the order of the contraction index is free as long as q is laid out alike;
//   V  a lane holds one word (eight columns) of four keys; cvt gives pairs of columns, two byte permutations pairs of keys.
// code x scale is exact in f16.  q is brought into f16's range by a power of two per row (exact for bf16; an fp32 row takes two columns, its
// upper and its lower 11 bits), P is scaled by 2^15 (the rest of f16's range) and, for fp32, split alike.  P^T comes out of the accumulators of
// S^T as the second product's other operand by a transposition within the warp (movmatrix).
//
// Each warp has a ring of its own of four key tiles, filled by untiled bulk copies (a tile is contiguous in each of the four tensors), and
// runs its softmax with nobody to wait for; W warps (and a cluster's `splits` blocks) share a unit, one (slot, key head, rows).
constexpr int MW = 4, NSTG = 4;
template <typename T, int HD, int NT> struct MmaShape {
  static constexpr int WORDS = HD / 8, NB = HD / BLOCK, WPT = (WORDS + 3) / 4, NWV = (WORDS + 7) / 8;
  static constexpr int TK = HD <= 64 ? 64 : 32, KS = NT == 1 ? TK : 32;         // keys of a tile; of one step of the softmax
  static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, ROWS = 8 * NT / PARTS;   // columns per row; rows of a unit
  static constexpr int CODE_BYTES = TK * HD / 2, SCALE_BYTES = TK * NB, STAGE = 2 * (CODE_BYTES + SCALE_BYTES);
  static constexpr int WARP_BYTES = NSTG * STAGE;
  static constexpr int SMEM = MW * WARP_BYTES + MW * NSTG * 8;
  static_assert(ROWS * (HD + 2) * 4 <= WARP_BYTES && STAGE % 16 == 0 && SCALE_BYTES % 16 == 0, "");
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
// the eight values of a word of codes as four f16x2
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) { uint32_t d; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) { uint32_t d; asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) { uint32_t d; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo)); return d; }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
constexpr float P_SHIFT = 15.f;                        // P <= 2^15

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(MW * 32) attention_kv4_mma_kernel(const Kv4Attn p, int log_w, int tiles) {
  using S = MmaShape<T, HD, NT>;
  constexpr int WPT = S::WPT, NWV = S::NWV, NB = S::NB, TK = S::TK, KS = S::KS, ROWS = S::ROWS, PARTS = S::PARTS, G16 = KS / 16;
  constexpr int CPL = PARTS == 1 ? 2 : 1;              // rows in a lane's two columns
  extern __shared__ __align__(128) unsigned char sm[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  const int W = 1 << log_w, wi = warp & (W - 1), split = blockIdx.x % p.splits;
  unsigned char* ring = sm + warp * S::WARP_BYTES;
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + MW * S::WARP_BYTES) + warp * NSTG;
  if (lane < NSTG) tc05::mbar_init(&bar[lane], 1);
  tc05::fence_barrier_init();
  __syncwarp();
  pdl_trigger();
  pdl_wait();
  const long long unit = (long long)(blockIdx.x / p.splits) * (MW >> log_w) + (warp >> log_w);
  const int tile = (int)(unit % tiles);
  const long long pair = unit / tiles;
  const int h = (int)(pair % p.d.heads), s = (int)(pair / p.d.heads);
  int len = 0, cnt = 0;
  if (s < p.d.slots) {
    len = min(max(p.lens[s], 0), p.d.capacity);
    cnt = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
  }
  const int r0 = tile * ROWS, rows = max(0, min(ROWS, cnt * p.group - r0));
  // keys that row r sees; the last row sees most
  auto sees = [&](int r) { return r < rows ? max(0, len - cnt + (r0 + r) / p.group + 1) : 0; };
  const int most = rows > 0 ? sees(rows - 1) : 0, least = sees(0);
  int see[NT][CPL];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < CPL; ++c) see[t][c] = sees(PARTS == 1 ? t * 8 + 2 * j + c : t * 4 + j);

  // ---- the ring: lane x knows the slot of the warp's x-th tile (of 32 at a time), lane 0 issues
  const int first = split * W + wi, step = p.splits * W, n_tiles = max(0, ceil_div(ceil_div(most, TK) - first, step));
  const unsigned char* kc0 = p.d.kc + p.layer * p.d.code_layer + (long long)h * p.d.capacity * (HD / 2);
  const unsigned char* vc0 = p.d.vc + p.layer * p.d.code_layer + (long long)h * p.d.capacity * (HD / 2);
  const unsigned char* ks0 = p.d.ks + p.layer * p.d.scale_layer + (long long)h * p.d.capacity * NB;
  const unsigned char* vs0 = p.d.vs + p.layer * p.d.scale_layer + (long long)h * p.d.capacity * NB;
  int slot_of = s, bad = 0;                            // bad: bit per stage, its page names no slot
  auto issue = [&](int i) {
    if (i % 32 == 0) {
      const int t = first + (i + lane) * step;
      slot_of = s;
      if (p.pages && t * TK < most) slot_of = p.pages[(long long)s * (p.d.capacity / PAGE) + t * TK / PAGE];
    }
    int slot = __shfl_sync(0xffffffffu, slot_of, i % 32);
    const int st = i % NSTG;
    bad &= ~(1 << st);
    if (slot < 0 || slot >= p.d.slots) { bad |= 1 << st; slot = s; }
    if (lane == 0) {
      unsigned char* dst = ring + st * S::STAGE;
      const long long t = first + (long long)i * step, co = slot * p.d.code_slot + t * S::CODE_BYTES, so = slot * p.d.scale_slot + t * S::SCALE_BYTES;
      tc05::mbar_expect_tx(&bar[st], S::STAGE);
      tc05::bulk_load_1d(dst, kc0 + co, S::CODE_BYTES, &bar[st]);
      tc05::bulk_load_1d(dst + S::CODE_BYTES, ks0 + so, S::SCALE_BYTES, &bar[st]);
      tc05::bulk_load_1d(dst + S::CODE_BYTES + S::SCALE_BYTES, vc0 + co, S::CODE_BYTES, &bar[st]);
      tc05::bulk_load_1d(dst + 2 * S::CODE_BYTES + S::SCALE_BYTES, vs0 + so, S::SCALE_BYTES, &bar[st]);
    }
  };
  for (int i = 0; i < min(NSTG, n_tiles); ++i) issue(i);

  // ---- q: lane (g, j) holds the words j WPT .. of column g, as f16 of q 2^-e; c of a lane's own columns brings the scores to log2 units
  uint32_t qf[NT][WPT][4];
  float cf[NT][CPL];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int col = t * 8 + g, r = PARTS == 1 ? col : col / 2;
    float x[WPT][8], amax = 0.f;
    const long long at = s * p.qb + (long long)((r0 + r) / p.group) * p.qt + (h * p.group + (r0 + r) % p.group) * p.qh;
#pragma unroll
    for (int i = 0; i < WPT; ++i) {
      const int w = j * WPT + i;
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        x[i][y] = r < rows && w < S::WORDS ? to_f<T>(reinterpret_cast<const T*>(p.q)[at + w * 8 + y]) : 0.f;
        amax = fmaxf(amax, fabsf(x[i][y]));
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = amax > 0.f && amax <= 3.402823466e38f ? ilogbf(amax) - 14 : 0;
#pragma unroll
    for (int i = 0; i < WPT; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float a = ldexpf(x[i][2 * y], -e), b = ldexpf(x[i][2 * y + 1], -e);
        const uint32_t hi = f16x2(a, b);
        const float2 back = f16x2_f32(hi);
        qf[t][i][y] = PARTS == 1 || (g & 1) == 0 ? hi : f16x2(a - back.x, b - back.y);
      }
    const float c = ldexpf(p.scale_log2, e + p.d.k_exp);
#pragma unroll
    for (int y = 0; y < CPL; ++y) cf[t][y] = __shfl_sync(0xffffffffu, c, 4 * (2 * j + y));
  }

  float o[NWV][4][NT][4], m[NT][CPL], l[NT][CPL];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) { m[t][c] = -INFINITY; l[t][c] = 0.f; }
#pragma unroll
    for (int i = 0; i < NWV; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[i][u][t][y] = 0.f;
  }
  const int kperm = (g >> 1) + 4 * (g & 1);            // the key of row g of a tile: the keys of a lane's two columns of P^T then lie four apart in V
  bool failed = false;
  for (int i = 0; i < n_tiles; ++i) {
    const int st = i % NSTG;
    if (!tc05::mbar_wait(&bar[st], (i / NSTG) & 1)) { failed = true; break; }
    const unsigned char *kc = ring + st * S::STAGE, *ks = kc + S::CODE_BYTES, *vc = ks + S::SCALE_BYTES, *vs = vc + S::CODE_BYTES;
    const int base0 = (first + i * step) * TK;
    const bool nan_tile = (bad >> st) & 1;
#pragma unroll
    for (int k0 = 0; k0 < TK; k0 += KS) {
      const int base = base0 + k0;
      if (k0 > 0 && base >= most) break;
      float sc[G16][NT][4];
#pragma unroll
      for (int a = 0; a < G16; ++a) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int y = 0; y < 4; ++y) sc[a][t][y] = 0.f;
        const int ka = k0 + a * 16 + kperm, kb = ka + 8;
        uint32_t sa = 0, sb = 0;
        uint32_t wa[WPT], wb[WPT];
        if constexpr (WPT == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(kc + ka * (HD / 2) + j * 8), y = *reinterpret_cast<const uint2*>(kc + kb * (HD / 2) + j * 8);
          wa[0] = x.x; wa[1] = x.y; wb[0] = y.x; wb[1] = y.y;
        } else if constexpr (WPT == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(kc + ka * (HD / 2) + j * 16), y = *reinterpret_cast<const uint4*>(kc + kb * (HD / 2) + j * 16);
          wa[0] = x.x; wa[1] = x.y; wa[2] = x.z; wa[3] = x.w; wb[0] = y.x; wb[1] = y.y; wb[2] = y.z; wb[3] = y.w;
        } else {
#pragma unroll
          for (int x = 0; x < WPT; ++x) {
            const int w = j * WPT + x;
            const bool in = S::WORDS % 4 == 0 || w < S::WORDS;
            wa[x] = in ? *reinterpret_cast<const uint32_t*>(kc + ka * (HD / 2) + w * 4) : 0u;
            wb[x] = in ? *reinterpret_cast<const uint32_t*>(kc + kb * (HD / 2) + w * 4) : 0u;
          }
        }
#pragma unroll
        for (int x = 0; x < WPT; ++x) {
          if (WPT % 2 == 1 || x % 2 == 0) {            // a new block of 16
            int blk = (j * WPT + x) >> 1;
            if (S::WORDS % 4 != 0) blk = min(blk, NB - 1);
            const uint32_t two = e4m3x2_f16x2(ks[ka * NB + blk] | (uint32_t)ks[kb * NB + blk] << 8);
            sa = __byte_perm(two, two, 0x1010); sb = __byte_perm(two, two, 0x3232);
          }
          uint32_t ha[4], hb[4];
          unpack8(wa[x], ha); unpack8(wb[x], hb);
#pragma unroll
          for (int y = 0; y < 4; ++y) { ha[y] = mul2(ha[y], sa); hb[y] = mul2(hb[y], sb); }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_16816(sc[a][t], ha[0], hb[0], ha[1], hb[1], qf[t][x][0], qf[t][x][1]);
            mma_16816(sc[a][t], ha[2], hb[2], ha[3], hb[3], qf[t][x][2], qf[t][x][3]);
          }
        }
      }
      // ---- softmax: sc[a][t][0], [1]: key kperm of group a, a lane's two columns; [2], [3]: key kperm + 8
      uint32_t pf[G16][NT][2];
      const bool masked = base + KS > least;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float mx[CPL];
#pragma unroll
        for (int c = 0; c < CPL; ++c) mx[c] = -INFINITY;
#pragma unroll
        for (int a = 0; a < G16; ++a) {
          float (&x)[4] = sc[a][t];
          if (PARTS == 2) { x[0] += x[1]; x[2] += x[3]; }
#pragma unroll
          for (int c = 0; c < CPL; ++c) {
            x[c] *= cf[t][c]; x[2 + c] *= cf[t][c];
            if (nan_tile) x[c] = x[2 + c] = __int_as_float(0x7fc00000);
            if (masked) {
              if (base + a * 16 + kperm >= see[t][c]) x[c] = -INFINITY;
              if (base + a * 16 + kperm + 8 >= see[t][c]) x[2 + c] = -INFINITY;
            }
            mx[c] = fmaxf(mx[c], fmaxf(x[c], x[2 + c]));
          }
        }
        bool moved = false;
        float al[CPL], ref[CPL];
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 4));
          mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 8));
          mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 16));
          const float mn = fmaxf(m[t][c], mx[c]), safe = mn == -INFINITY ? 0.f : mn;
          al[c] = ex2(m[t][c] - safe);
          moved |= mn != m[t][c];
          ref[c] = safe - P_SHIFT;
          m[t][c] = mn;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int c = 0; c < CPL; ++c) l[t][c] *= al[c];
#pragma unroll
          for (int x = 0; x < NWV; ++x)
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int y = 0; y < 4; ++y) o[x][u][t][y] *= al[y % CPL];
        }
#pragma unroll
        for (int a = 0; a < G16; ++a) {
          float (&x)[4] = sc[a][t];
          uint32_t lo, hi;
          if (PARTS == 1) {
            const float p0 = ex2(x[0] - ref[0]), p1 = ex2(x[1] - ref[CPL - 1]), p2 = ex2(x[2] - ref[0]), p3 = ex2(x[3] - ref[CPL - 1]);
            l[t][0] += p0 + p2; l[t][CPL - 1] += p1 + p3;
            lo = f16x2(p0, p1); hi = f16x2(p2, p3);
          } else {
            const float p0 = ex2(x[0] - ref[0]), p2 = ex2(x[2] - ref[0]);
            l[t][0] += p0 + p2;
            const float2 r = f16x2_f32(f16x2(p0, p2));
            lo = f16x2(p0, p0 - r.x); hi = f16x2(p2, p2 - r.y);
          }
          pf[a][t][0] = transpose8(lo); pf[a][t][1] = transpose8(hi);
        }
      }
      // ---- o^T += V^T P^T
#pragma unroll
      for (int a = 0; a < G16; ++a) {
        const int kv = k0 + a * 16 + j;                // this lane's keys: kv, + 4, + 8, + 12
#pragma unroll
        for (int x = 0; x < NWV; ++x) {
          const int w = g + 8 * x;
          const bool in = S::WORDS % 8 == 0 || w < S::WORDS;
          const int ws = in ? w : 0;
          uint32_t hv[4][4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(vc + (kv + 4 * y) * (HD / 2) + ws * 4);
            unpack8(in ? word : 0u, hv[y]);
          }
          const unsigned char* f = vs + kv * NB + (ws >> 1);
          // A NaN scale becomes 448 here: the key's scales are NaN as well and say so to the rows that see it, and to no other.  The same makes
          // whatever lies behind the last token a number, which its zero weight removes.
          const uint32_t s01 = min2(e4m3x2_f16x2(f[0] | (uint32_t)f[4 * NB] << 8), 0x5f005f00u), s23 = min2(e4m3x2_f16x2(f[8 * NB] | (uint32_t)f[12 * NB] << 8), 0x5f005f00u);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t a0 = mul2(__byte_perm(hv[0][u], hv[1][u], 0x5410), s01), a1 = mul2(__byte_perm(hv[0][u], hv[1][u], 0x7632), s01);
            const uint32_t a2 = mul2(__byte_perm(hv[2][u], hv[3][u], 0x5410), s23), a3 = mul2(__byte_perm(hv[2][u], hv[3][u], 0x7632), s23);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_16816(o[x][u][t], a0, a1, a2, a3, pf[a][t][0], pf[a][t][1]);
          }
        }
      }
    }
    __syncwarp();                                      // every lane has read the stage
    if (i + NSTG < n_tiles) issue(i + NSTG);
  }
  if (failed) {                                        // leave with no copy in flight
    if (lane == 0) atomicExch(p.status, LLMB_ERR_TIMEOUT);
    for (int st = 0; st < NSTG; ++st) tc05::mbar_wait(&bar[st], 0);
  }
  // ---- partial results: rows of HD sums, then maxima, then row sums, where the warp's ring was
  float* po = reinterpret_cast<float*>(ring);
  float *pm = po + ROWS * HD, *pl = pm + ROWS;
  __syncwarp();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      float v = l[t][c];
      v += __shfl_xor_sync(0xffffffffu, v, 4); v += __shfl_xor_sync(0xffffffffu, v, 8); v += __shfl_xor_sync(0xffffffffu, v, 16);
      const int r = PARTS == 1 ? t * 8 + 2 * j + c : t * 4 + j;
      if (g == 0) { pm[r] = m[t][c]; pl[r] = v; }
#pragma unroll
      for (int x = 0; x < NWV; ++x)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int w = g + 8 * x;
          if (r < rows && (S::WORDS % 8 == 0 || w < S::WORDS)) {
            float2 v2;
            if (PARTS == 1) v2 = make_float2(o[x][u][t][c], o[x][u][t][2 + c]);
            else v2 = make_float2(o[x][u][t][0] + o[x][u][t][1], o[x][u][t][2] + o[x][u][t][3]);
            *reinterpret_cast<float2*>(po + r * HD + w * 8 + 2 * u) = v2;
          }
        }
    }
  }
  if (W > 1) __syncthreads(); else __syncwarp();
  const float vunit = pow2(p.d.v_exp);
  constexpr int PITCH = S::WARP_BYTES / 4;             // floats between two warps' parts
  float* u0 = reinterpret_cast<float*>(sm + (warp & ~(W - 1)) * S::WARP_BYTES);
  auto store = [&](int r, int c, float sum, float total) {
    const long long at = s * p.ob + (long long)((r0 + r) / p.group) * p.ot + (h * p.group + (r0 + r) % p.group) * p.oh + c;
    reinterpret_cast<T*>(p.out)[at] = from_f<T>(total == 0.f ? 0.f : sum / total * vunit);
  };
  if (p.splits == 1) {
    for (int x = wi * 32 + lane; x < rows * HD; x += W * 32) {
      const int r = x / HD, c = x % HD;
      float mx = -INFINITY, sum = 0.f, total = 0.f;
      for (int w = 0; w < W; ++w) mx = fmaxf(mx, u0[w * PITCH + ROWS * HD + r]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      for (int w = 0; w < W; ++w) {
        const float f = ex2(u0[w * PITCH + ROWS * HD + r] - ref);
        sum += u0[w * PITCH + x] * f; total += u0[w * PITCH + ROWS * HD + ROWS + r] * f;
      }
      store(r, c, sum, total);
    }
    return;
  }
  // a cluster per unit (W = MW): each block leaves its parts as they are, and finishes a share of the elements from everybody's
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int x = split * (MW * 32) + threadIdx.x; x < rows * HD; x += p.splits * MW * 32) {
    const int r = x / HD, c = x % HD;
    float mx = -INFINITY, sum = 0.f, total = 0.f;
    for (int k = 0; k < p.splits; ++k) {
      const float* u = cluster.map_shared_rank(u0, k);
      for (int w = 0; w < MW; ++w) mx = fmaxf(mx, u[w * PITCH + ROWS * HD + r]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx;
    for (int k = 0; k < p.splits; ++k) {
      const float* u = cluster.map_shared_rank(u0, k);
      for (int w = 0; w < MW; ++w) {
        const float f = ex2(u[w * PITCH + ROWS * HD + r] - ref);
        sum += u[w * PITCH + x] * f; total += u[w * PITCH + ROWS * HD + ROWS + r] * f;
      }
    }
    store(r, c, sum, total);
  }
  cluster.sync();                                      // no block leaves while another reads its shared memory
}

inline int allow_smem(unsigned long long& done, const void* kernel, int bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < 64 && (done >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done |= 1ull << dev;
  }
  return (int)e;
}

template <typename T, int HD, int NT>
int run_mma(Kv4Attn p, cudaStream_t st) {
  using S = MmaShape<T, HD, NT>;
  static unsigned long long attr = 0;                  // devices on which the kernel may take its shared memory
  if (const int e = allow_smem(attr, (const void*)attention_kv4_mma_kernel<T, HD, NT>, S::SMEM)) return e;
  const long long tiles = ceil_div_ll((long long)p.n * p.group, S::ROWS), units = tiles * p.d.heads * p.d.slots;
  // One warp a unit where there are enough of them to fill the chip (three blocks of four warps on an SM), else two, four, and a cluster.
  const long long want = (long long)sm_count() * 12;
  const int most = ceil_div(p.d.capacity, S::TK);      // no more warps than tiles
  int log_w = 0;
  while (log_w < 2 && (units << log_w) < want && (1 << log_w) < most) ++log_w;
  p.splits = 1;
  if (log_w == 2) while (p.splits < 8 && units * 4 * p.splits < want && p.splits * 4 < most) p.splits *= 2;
  const long long blocks = ceil_div_ll(units << log_w, MW) * p.splits;
  if (blocks > 0x7fffffffLL || tiles > 0x7fffffffLL) return LLMB_ERR_BAD_ARG;
  return launch_pdl_cluster(dim3(p.splits), attention_kv4_mma_kernel<T, HD, NT>, dim3((unsigned)blocks), MW * 32, S::SMEM, st, p, log_w, (int)tiles);
}
template <typename T, int HD>
int run(const Kv4Attn& p, cudaStream_t st) {
  const long long rows = (long long)p.n * p.group;
  constexpr int R8 = sizeof(T) == 4 ? 4 : 8, MOST = HD <= 64 ? 4 : 2;
  if (rows <= R8) return run_mma<T, HD, 1>(p, st);
  if (rows <= 2 * R8 || MOST == 2) return run_mma<T, HD, 2>(p, st);
  return run_mma<T, HD, MOST>(p, st);
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

// The arguments of a call as the Python side (ops/kv4.py) packs them.
struct Kv4AttendArgs {
  void* out; const void* q; const int *lens, *counts, *pages;   // counts, pages: optional
  int* status;
  long long qb, qt, qh, ob, ot, oh;
  float scale;
  int layer, n, heads, dtype, pad;
};

LLMB_API int llmb_attention_kv4(const Kv4Desc* d, const Kv4AttendArgs* a, cudaStream_t st) {
  if (a->heads % d->heads) return LLMB_ERR_BAD_ARG;
  Kv4Attn p{*d, a->out, a->q, a->lens, a->counts, a->pages, a->layer, a->n, a->heads / d->heads, 1, a->scale * 1.4426950408889634f,
            a->qb, a->qt, a->qh, a->ob, a->ot, a->oh, a->status};
  return a->dtype == LLMB_BF16 ? run_type<__nv_bfloat16>(p, st) : run_type<float>(p, st);
}
