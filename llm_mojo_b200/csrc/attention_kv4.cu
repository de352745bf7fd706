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
// The products are taken transposed, S^T = K q^T and o^T = V^T P^T (mma.sync m16n8k16, f16 operands, fp32 sums): 16 keys fill a tile's rows
// and eight columns are rows of q, so that a single query pads to 8 and not to 128 (as it would in a tcgen05 product), and the codes
// go from shared memory to registers straight into operands:
//   K  a lane holds contiguous words of a key's row; the order of the contraction index is free as long as q is laid out alike;
//   V  a lane holds one word (eight columns) of four keys; of the words behind a multiple of eight, a half or
//      a quarter (64 x 16 heads of 80, up to 1024 tokens: 30.2 us with whole words, 27.9 so).  cvt turns a byte into a pair of columns of one key, but the contraction runs over
//      keys.  With few rows (NARROW: two columns of the tile per row) the pair is contracted as it stands, against (p, 0) in a row's
//      first column, which gives the even columns of o, and (0, p) in its second, the odd ones; with more rows two byte permutations
//      of every four values make pairs of keys.
// code x scale is exact in f16.  q is brought into f16's range by a power of two per row (exact for bf16; an fp32 row takes two columns, its
// upper and its lower 11 bits), P is scaled by a power of two into the rest of f16's range and, for fp32, split alike.  In bf16 a weight is so off by
// up to 2^-11 of itself, an eighth of what the result's own rounding is (one below f16's normal numbers by 2^-32 of their sum); the sum that it is
// divided by is taken of the fp32 weights.  P^T comes out of the accumulators of
// S^T as the second product's other operand by a transposition within the warp (movmatrix).
//
// Each warp has a ring of its own of key tiles, filled by untiled bulk copies (a tile is contiguous in each of the four tensors), and
// runs its softmax with nobody to wait for; W warps (and a cluster's `splits` blocks) share a unit, one (slot, key head, rows).
constexpr int NSTG = 2, MOST_WARPS = 8, MOST_SPLITS = 16;
template <typename T, int HD, int NT, bool NARROW> struct MmaShape {
  static constexpr int WORDS = HD / 8, NB = HD / BLOCK, WPT = (WORDS + 3) / 4, NWV = (WORDS + 7) / 8;
  static constexpr int TAIL = WORDS % 8 / 2;           // bytes of V that a lane takes where eight lanes have no word each: heads of 80, and of 32 and 96
  // keys of a tile: as many as two stages of shared memory hold for the warps of an SM (heads of 80: 27.9 us with 32, 25.8); of one step of the softmax
  static constexpr int TK = HD <= 96 ? 64 : 32, KS = NT == 1 ? TK : 32;
  static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, PER_ROW = PARTS * (NARROW ? 2 : 1), ROWS = 8 * NT / PER_ROW;   // columns per row; rows of a unit
  static constexpr int CODE_BYTES = TK * HD / 2, SCALE_BYTES = TK * NB, STAGE = 2 * (CODE_BYTES + SCALE_BYTES);
  static constexpr int WARP_BYTES = NSTG * STAGE;
  static constexpr int SMEM_WARP = WARP_BYTES + NSTG * 8;
  static constexpr int WARPS_SM = NT > 2 || (NT == 2 && HD > 64) ? 8 : NT == 2 ? 12 : HD <= 64 ? 24 : 16;             // registers decide
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
__device__ __forceinline__ uint32_t low2(uint32_t a) { uint32_t d; asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tmov.b32 %0, {l, l};\n\t}" : "=r"(d) : "r"(a)); return d; }
__device__ __forceinline__ uint32_t high2(uint32_t a) { uint32_t d; asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tmov.b32 %0, {h, h};\n\t}" : "=r"(d) : "r"(a)); return d; }
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) { uint32_t d; asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) { uint32_t d; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo)); return d; }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
constexpr float P_TOP = 15.f, LAG = 8.f;               // P <= 2^15; with one tile of columns the maximum may lag by 2^8

template <typename T, int HD, int NT, bool NARROW>
__global__ void __launch_bounds__(MOST_WARPS * 32, MmaShape<T, HD, NT, NARROW>::WARPS_SM / MOST_WARPS)
attention_kv4_mma_kernel(const Kv4Attn p, int log_w, int tiles) {
  using S = MmaShape<T, HD, NT, NARROW>;
  constexpr int WPT = S::WPT, NWV = S::NWV, NB = S::NB, TK = S::TK, KS = S::KS, ROWS = S::ROWS, PARTS = S::PARTS, PER_ROW = S::PER_ROW, G16 = KS / 16;
  constexpr int CPL = PER_ROW == 1 ? 2 : 1;            // rows in a lane's two columns
  constexpr int NO = NARROW ? 2 : 4;                   // accumulator tiles of o^T per word of V
  static_assert(!NARROW || NT == 1, "");
  extern __shared__ __align__(128) unsigned char sm[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  const int MW = blockDim.x / 32, W = 1 << log_w, wi = warp & (W - 1), split = p.splits == 1 ? 0 : blockIdx.x % p.splits;
  unsigned char* ring = sm + warp * S::WARP_BYTES;
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + MW * S::WARP_BYTES) + warp * NSTG;
  if (lane < NSTG) tc05::mbar_init(&bar[lane], 1);
  tc05::fence_barrier_init();
  __syncwarp();
  pdl_trigger();
  pdl_wait();
  const int unit = (p.splits == 1 ? blockIdx.x : blockIdx.x / p.splits) * (MW >> log_w) + (warp >> log_w);
  const int tile = tiles == 1 ? 0 : unit % tiles, pair = tiles == 1 ? unit : unit / tiles;
  const int s = pair / p.d.heads, h = pair - s * p.d.heads;
  const bool here = s < p.d.slots;

  // ---- the ring: lanes 0 .. 3 issue the copies of a tile, one each: key codes, key scales, value codes, value scales.  Lane x knows the
  // slot of the warp's x-th tile (of 32 at a time).  The first tile is fetched before the length is known: it lies in the cache in any case.
  const int first = split * W + wi, step = p.splits * W, cap_tiles = p.d.capacity / TK;
  const unsigned char* src = lane == 0 ? p.d.kc : lane == 1 ? p.d.ks : lane == 2 ? p.d.vc : p.d.vs;
  const int piece = lane & 1 ? S::SCALE_BYTES : S::CODE_BYTES;
  const long long src_slot = lane & 1 ? p.d.scale_slot : p.d.code_slot;
  const uint32_t dst = tc05::smem_u32(ring) + (lane & 1 ? S::CODE_BYTES : 0) + (lane & 2 ? S::CODE_BYTES + S::SCALE_BYTES : 0);
  src += p.layer * (lane & 1 ? p.d.scale_layer : p.d.code_layer) + (long long)h * cap_tiles * piece;
  int slot_of = s, bad = 0;                            // bad: bit per stage, its page names no slot
  const unsigned char* next_src = src + s * src_slot + (long long)first * piece;          // of the warp's next tile, in its own slot
  const long long hop = (long long)step * piece;
  auto issue = [&](int i) {
    const int st = i % NSTG;
    const unsigned char* from = next_src;
    next_src += hop;
    if (p.pages) {
      if (i % 32 == 0) {
        const int t = first + (i + lane) * step;
        slot_of = t < cap_tiles ? p.pages[(long long)s * (p.d.capacity / PAGE) + t * TK / PAGE] : s;
      }
      int slot = __shfl_sync(0xffffffffu, slot_of, i % 32);
      bad &= ~(1 << st);
      if (slot < 0 || slot >= p.d.slots) { bad |= 1 << st; slot = s; }
      from += (slot - s) * src_slot;
    }
    if (lane == 0) tc05::mbar_expect_tx(&bar[st], S::STAGE);
    __syncwarp();
    if (lane < 4)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   ::"r"(dst + st * S::STAGE), "l"(from), "r"(piece), "r"(tc05::smem_u32(&bar[st])) : "memory");
  };
  const bool early = here && first < cap_tiles;
  if (early) issue(0);
  int len = 0, cnt = 0;
  if (here) {
    len = min(max(p.lens[s], 0), p.d.capacity);
    cnt = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
  }
  const int r0 = tile * ROWS, rows = max(0, min(ROWS, cnt * p.group - r0));
  // keys that row r sees; the last row sees most
  auto token_of = [&](int r) { return p.n == 1 ? 0 : p.group == 1 ? r0 + r : (r0 + r) / p.group; };
  auto sees = [&](int r) { return r < rows ? max(0, len - cnt + token_of(r) + 1) : 0; };
  auto row_of = [&](int t, int c) { return PER_ROW == 1 ? t * 8 + 2 * j + c : PER_ROW == 2 ? t * 4 + j : j >> 1; };     // of this lane's columns
  const int most = rows > 0 ? sees(rows - 1) : 0, least = sees(0);
  int see[NT][CPL];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < CPL; ++c) see[t][c] = sees(row_of(t, c));
  const int n_tiles = max(0, ceil_div(ceil_div(most, TK) - first, step));
  for (int i = 1; i < min(NSTG, n_tiles); ++i) issue(i);

  // ---- q: lane (g, j) holds the words j WPT .. of column g, as f16 of q 2^-e; c of a lane's own columns brings the scores to log2 units.  c is
  // positive (the scale's sign goes to q; without a scale all scores are 0), so the largest score is the largest product.
  uint32_t qf[NT][WPT][4];
  float cf[NT][CPL];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = t * (8 / PER_ROW) + g / PER_ROW;
    float x[WPT][8], amax = 0.f;
    const int token = token_of(r);
    const T* q = reinterpret_cast<const T*>(p.q) + (s * p.qb + token * p.qt + (h * p.group + r0 + r - token * p.group) * p.qh + j * WPT * 8);
#pragma unroll
    for (int i = 0; i < WPT; ++i) {
#pragma unroll
      for (int y = 0; y < 8; ++y) x[i][y] = 0.f;
      if (r < rows && j * WPT + i < S::WORDS) {
        if (p.q_vec) {
#pragma unroll
          for (int y = 0; y < 8 / Pack<T>::N; ++y) {
            Pack<T> v; v.load(q + i * 8 + y * Pack<T>::N);
#pragma unroll
            for (int z = 0; z < Pack<T>::N; ++z) x[i][y * Pack<T>::N + z] = v.v[z];
          }
        } else {
#pragma unroll
          for (int y = 0; y < 8; ++y) x[i][y] = to_f<T>(q[i * 8 + y]);
        }
      }
#pragma unroll
      for (int y = 0; y < 8; ++y) amax = fmaxf(amax, fabsf(x[i][y]));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // amax 2^-e lies in [2^14, 2^15); a row without a value of 2^-86 or more has no score of any size
    const int e = max((int)(__float_as_uint(amax) >> 23) - 141, -100);
    const float down = amax <= 3.402823466e38f ? (p.scale_log2 < 0.f ? -1.f : p.scale_log2 == 0.f ? 0.f : 1.f) * pow2(-e) : __int_as_float(0x7fc00000);
#pragma unroll
    for (int i = 0; i < WPT; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float a = x[i][2 * y] * down, b = x[i][2 * y + 1] * down;
        const uint32_t hi = f16x2(a, b);
        const float2 back = f16x2_f32(hi);
        qf[t][i][y] = PARTS == 1 || (g & 1) == 0 ? hi : f16x2(a - back.x, b - back.y);
      }
    const float c = p.scale_log2 == 0.f ? 1.f : fmaxf(fabsf(p.scale_log2) * pow2(e / 2) * pow2(e - e / 2) * pow2(p.d.k_exp), 1e-37f);
#pragma unroll
    for (int y = 0; y < CPL; ++y) cf[t][y] = __shfl_sync(0xffffffffu, c, 4 * (2 * j + y));
  }

  // m: the reference maximum of the products, not yet times c; ref: what is added to the products times c; lag: how far they may pass m
  constexpr float SHIFT = NT == 1 ? P_TOP - LAG : P_TOP;
  float o[NWV][NO][NT][4], m[NT][CPL], l[NT][CPL], ref[NT][CPL], lag[NT][CPL];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) { m[t][c] = -INFINITY; l[t][c] = 0.f; ref[t][c] = SHIFT; lag[t][c] = NT == 1 ? LAG / cf[t][c] : 0.f; }
#pragma unroll
    for (int i = 0; i < NWV; ++i)
#pragma unroll
      for (int u = 0; u < NO; ++u)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[i][u][t][y] = 0.f;
  }
  auto bytes_of = [](int x) { return S::TAIL && x == NWV - 1 ? S::TAIL : 4; };          // of the x-th piece of a row of V, and where they lie
  auto first_byte = [g](int x) { return 32 * x + (S::TAIL && x == NWV - 1 ? S::TAIL : 4) * g; };
  const int kperm = (g >> 1) + 4 * (g & 1);            // the key of row g of a tile: the keys of a lane's two columns of P^T then lie four apart in V
  const uint32_t sel_a = g & 1 ? 0x1044 : 0x4410, sel_b = g & 1 ? 0x3244 : 0x4432;      // NARROW: (p, 0) or (0, p) of the lower and the upper half
  int failed_at = -1;
  for (int i = 0; i < n_tiles; ++i) {
    const int st = i % NSTG;
    if (!tc05::mbar_wait(&bar[st], (i / NSTG) & 1)) { failed_at = i; break; }
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
            sa = low2(two); sb = high2(two);
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
      // ---- softmax: sc[a][t][0], [1]: key kperm of group a, a lane's two columns; [2], [3]: key kperm + 8.  Where the two columns belong to one
      // row, [0] and [2] are brought to hold its scores.
      if (PARTS == 2) {
#pragma unroll
        for (int a = 0; a < G16; ++a)
#pragma unroll
          for (int t = 0; t < NT; ++t) { sc[a][t][0] += sc[a][t][1]; sc[a][t][2] += sc[a][t][3]; }
      }
      if (nan_tile) {
#pragma unroll
        for (int a = 0; a < G16; ++a)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int y = 0; y < 4; ++y) sc[a][t][y] = __int_as_float(0x7fc00000);
      }
      if (base + KS > least) {
#pragma unroll
        for (int a = 0; a < G16; ++a)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < CPL; ++c) {
              if (base + a * 16 + kperm >= see[t][c]) sc[a][t][c] = -INFINITY;
              if (base + a * 16 + kperm + 8 >= see[t][c]) sc[a][t][2 + c] = -INFINITY;
            }
      }
      uint32_t pf[G16][NT][NARROW ? 4 : 2];            // NARROW: the two operands of the lower eight keys, then of the upper
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float mx[CPL];
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          mx[c] = fmaxf(sc[0][t][c], sc[0][t][2 + c]);
#pragma unroll
          for (int a = 1; a < G16; ++a) mx[c] = fmaxf(mx[c], fmaxf(sc[a][t][c], sc[a][t][2 + c]));
        }
        // A lane's own maximum says whether the reference has to move: mostly it has not, and the exchange and the rescaling are left out.
        bool move = mx[0] > m[t][0] + lag[t][0];
        if (CPL == 2) move |= mx[CPL - 1] > m[t][CPL - 1] + lag[t][CPL - 1];
        if (__any_sync(0xffffffffu, move)) {
          float al[CPL];
#pragma unroll
          for (int c = 0; c < CPL; ++c) {
            mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 4));
            mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 8));
            mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 16));
            const float mn = fmaxf(m[t][c], mx[c]), safe = mn == -INFINITY ? 0.f : mn;
            al[c] = ex2((m[t][c] - safe) * cf[t][c]);
            ref[t][c] = SHIFT - safe * cf[t][c];
            m[t][c] = mn;
            l[t][c] *= al[c];
          }
#pragma unroll
          for (int x = 0; x < NWV; ++x)
#pragma unroll
            for (int u = 0; u < NO; ++u)
#pragma unroll
              for (int y = 0; y < 4; ++y) o[x][u][t][y] *= al[y % CPL];
        }
#pragma unroll
        for (int a = 0; a < G16; ++a) {
          const float (&x)[4] = sc[a][t];
          uint32_t lo, hi;
          if (CPL == 2) {
            const float2 c2 = make_float2(cf[t][0], cf[t][CPL - 1]), r2 = make_float2(ref[t][0], ref[t][CPL - 1]);
            const float2 u = __ffma2_rn(make_float2(x[0], x[1]), c2, r2), v = __ffma2_rn(make_float2(x[2], x[3]), c2, r2);
            const float p0 = ex2(u.x), p1 = ex2(u.y), p2 = ex2(v.x), p3 = ex2(v.y);
            l[t][0] += p0 + p2; l[t][CPL - 1] += p1 + p3;
            lo = f16x2(p0, p1); hi = f16x2(p2, p3);
          } else {
            const float p0 = ex2(fmaf(x[0], cf[t][0], ref[t][0])), p2 = ex2(fmaf(x[2], cf[t][0], ref[t][0]));
            l[t][0] += p0 + p2;
            if (PARTS == 1) { lo = f16x2(p0, p0); hi = f16x2(p2, p2); }
            else {
              const float2 r = f16x2_f32(f16x2(p0, p2));
              const float q0 = p0 - r.x, q2 = p2 - r.y;
              if (!NARROW) { lo = f16x2(p0, q0); hi = f16x2(p2, q2); }
              else { lo = j & 1 ? f16x2(q0, q0) : f16x2(p0, p0); hi = j & 1 ? f16x2(q2, q2) : f16x2(p2, p2); }
            }
          }
          lo = transpose8(lo); hi = transpose8(hi);
          if (!NARROW) { pf[a][t][0] = lo; pf[a][t][1] = hi; }
          else {
            pf[a][t][0] = __byte_perm(lo, 0, sel_a); pf[a][t][1] = __byte_perm(lo, 0, sel_b);
            pf[a][t][NARROW ? 2 : 0] = __byte_perm(hi, 0, sel_a); pf[a][t][NARROW ? 3 : 0] = __byte_perm(hi, 0, sel_b);
          }
        }
      }
      // ---- o^T += V^T P^T
#pragma unroll
      for (int a = 0; a < G16; ++a) {
        const int kv = k0 + a * 16 + j;                // this lane's keys: kv, + 4, + 8, + 12
#pragma unroll
        for (int x = 0; x < NWV; ++x) {
          const int nu = bytes_of(x), b0 = first_byte(x);
          uint32_t hv[4][4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const unsigned char* at = vc + (kv + 4 * y) * (HD / 2) + b0;
            if (nu == 4) unpack8(*reinterpret_cast<const uint32_t*>(at), hv[y]);
            else {
              const uint32_t bytes = nu == 2 ? *reinterpret_cast<const uint16_t*>(at) : *at;
              hv[y][0] = e2m1x2_f16x2(bytes & 0xff);
              hv[y][1] = nu == 2 ? e2m1x2_f16x2(bytes >> 8) : 0u;
              hv[y][2] = hv[y][3] = 0u;
            }
          }
          const unsigned char* f = vs + kv * NB + (b0 >> 3);
          // A NaN scale becomes 448 here: the key's scales are NaN as well and say so to the rows that see it, and to no other.  The same makes
          // whatever lies behind the last token a number, which its zero weight removes.
          const uint32_t s01 = min2(e4m3x2_f16x2(f[0] | (uint32_t)f[4 * NB] << 8), 0x5f005f00u), s23 = min2(e4m3x2_f16x2(f[8 * NB] | (uint32_t)f[12 * NB] << 8), 0x5f005f00u);
          if (NARROW) {
            const uint32_t sf[4] = {low2(s01), high2(s01), low2(s23), high2(s23)};
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (u < nu) hv[y][u] = mul2(hv[y][u], sf[y]);
#pragma unroll
            for (int u = 0; u < NO; ++u) {
              if (2 * u >= nu) continue;
              mma_16816(o[x][u][0], hv[0][2 * u & 3], hv[0][(2 * u + 1) & 3], hv[1][2 * u & 3], hv[1][(2 * u + 1) & 3], pf[a][0][0], pf[a][0][1]);
              mma_16816(o[x][u][0], hv[2][2 * u & 3], hv[2][(2 * u + 1) & 3], hv[3][2 * u & 3], hv[3][(2 * u + 1) & 3], pf[a][0][NARROW ? 2 : 0], pf[a][0][NARROW ? 3 : 0]);
            }
          } else {
#pragma unroll
            for (int u = 0; u < NO; ++u) {
              if (u >= nu) continue;
              const uint32_t a0 = mul2(__byte_perm(hv[0][u], hv[1][u], 0x5410), s01), a1 = mul2(__byte_perm(hv[0][u], hv[1][u], 0x7632), s01);
              const uint32_t a2 = mul2(__byte_perm(hv[2][u], hv[3][u], 0x5410), s23), a3 = mul2(__byte_perm(hv[2][u], hv[3][u], 0x7632), s23);
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_16816(o[x][u][t], a0, a1, a2, a3, pf[a][t][0], pf[a][t][1]);
            }
          }
        }
      }
    }
    __syncwarp();                                      // every lane has read the stage
    if (i + NSTG < n_tiles) issue(i + NSTG);
  }
  if (failed_at >= 0) {                                // leave with no copy in flight
    if (lane == 0) atomicExch(p.status, LLMB_ERR_TIMEOUT);
    for (int i = failed_at; i < min(n_tiles, failed_at + NSTG); ++i) tc05::mbar_wait(&bar[i % NSTG], (i / NSTG) & 1);
  }
  if (early && n_tiles == 0 && !tc05::mbar_wait(&bar[0], 0) && lane == 0) atomicExch(p.status, LLMB_ERR_TIMEOUT);
  // ---- partial results: rows of HD sums, then maxima (in log2 units), then row sums, where the warp's ring was
  float* po = reinterpret_cast<float*>(ring);
  float *pm = po + ROWS * HD, *pl = pm + ROWS;
  __syncwarp();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      float v = l[t][c];
      v += __shfl_xor_sync(0xffffffffu, v, 4); v += __shfl_xor_sync(0xffffffffu, v, 8); v += __shfl_xor_sync(0xffffffffu, v, 16);
      const int r = row_of(t, c);
      const bool mine = PER_ROW < 4 || (j & 1) == 0;   // PER_ROW 4: two lanes hold a row's two parts
      if (g == 0 && mine) { pm[r] = m[t][c] * cf[t][c]; pl[r] = v; }
#pragma unroll
      for (int x = 0; x < NWV; ++x) {
        const int nu = bytes_of(x);
        const bool in = r < rows;
        float* at = po + r * HD + 2 * first_byte(x);
#pragma unroll
        for (int u = 0; u < NO; ++u) {
          if ((NARROW ? 2 * u : u) >= nu) continue;
          const float (&y)[4] = o[x][u][t];
          if (NARROW) {                                // a byte's two columns, then the next byte's
            float4 v4 = make_float4(y[0], y[1], y[2], y[3]);
            if (PARTS == 2) {
              v4.x += __shfl_xor_sync(0xffffffffu, v4.x, 1); v4.y += __shfl_xor_sync(0xffffffffu, v4.y, 1);
              v4.z += __shfl_xor_sync(0xffffffffu, v4.z, 1); v4.w += __shfl_xor_sync(0xffffffffu, v4.w, 1);
            }
            if (in && mine && nu == 1) *reinterpret_cast<float2*>(at) = make_float2(v4.x, v4.y);
            else if (in && mine) *reinterpret_cast<float4*>(at + 4 * u) = v4;
          } else if (in) {
            *reinterpret_cast<float2*>(at + 2 * u) = PARTS == 1 ? make_float2(y[c], y[2 + c]) : make_float2(y[0] + y[1], y[2] + y[3]);
          }
        }
      }
    }
  }
  // Joining: what each warp's part of a row counts for, then four columns per lane.  For one block per unit that is the result; a cluster's blocks
  // (a unit each: W is the whole block) leave the sums of their warps in place of warp 0's part.
  __shared__ float part[MOST_WARPS][ROWS], um[ROWS], ul[ROWS], share[MOST_SPLITS][ROWS];
  constexpr int PITCH = S::WARP_BYTES / 4;             // floats between two warps' parts
  const int w0 = warp & ~(W - 1);
  float* u0 = reinterpret_cast<float*>(sm + w0 * S::WARP_BYTES);
  auto together = [&]() { if (W > 1) __syncthreads(); else __syncwarp(); };
  together();
  const float vunit = pow2(p.d.v_exp);
  for (int x = wi * 32 + lane; x < rows * W; x += W * 32) {
    const int r = x >> log_w, w = x & (W - 1);
    float mx = -INFINITY, total = 0.f;
    for (int y = 0; y < W; ++y) mx = fmaxf(mx, u0[y * PITCH + ROWS * HD + r]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    for (int y = 0; y < W; ++y) total += u0[y * PITCH + ROWS * HD + ROWS + r] * ex2(u0[y * PITCH + ROWS * HD + r] - ref);
    const float f = ex2(u0[w * PITCH + ROWS * HD + r] - ref);
    part[w0 + w][r] = p.splits > 1 ? f : total == 0.f ? 0.f : f / total * vunit;
    if (w == 0 && p.splits > 1) { um[r] = mx; ul[r] = total; }
  }
  together();
  auto store = [&](int r, int c, float4 v) {
    const int token = token_of(r);
    T* at = reinterpret_cast<T*>(p.out) + (s * p.ob + token * p.ot + (h * p.group + r0 + r - token * p.group) * p.oh + c);
    if (!p.o_vec) { at[0] = from_f<T>(v.x); at[1] = from_f<T>(v.y); at[2] = from_f<T>(v.z); at[3] = from_f<T>(v.w); }
    else if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(at) = v;
    else {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  };
  for (int x = wi * 32 + lane; x < rows * (HD / 4); x += W * 32) {
    const int r = x / (HD / 4), c = x % (HD / 4) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < W; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(u0 + w * PITCH + r * HD + c);
      const float f = part[w0 + w][r];
      sum.x += v.x * f; sum.y += v.y * f; sum.z += v.z * f; sum.w += v.w * f;
    }
    if (p.splits == 1) store(r, c, sum);
    else *reinterpret_cast<float4*>(u0 + r * HD + c) = sum;
  }
  if (p.splits == 1) return;
  // The blocks of a cluster: each finishes a share of the elements from everybody's.
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int x = threadIdx.x; x < rows * p.splits; x += blockDim.x) {
    const int r = x / p.splits, k = x % p.splits;
    float mx = -INFINITY, total = 0.f;
    for (int y = 0; y < p.splits; ++y) mx = fmaxf(mx, *cluster.map_shared_rank(&um[r], y));
    const float ref = mx == -INFINITY ? 0.f : mx;
    for (int y = 0; y < p.splits; ++y) total += *cluster.map_shared_rank(&ul[r], y) * ex2(*cluster.map_shared_rank(&um[r], y) - ref);
    share[k][r] = total == 0.f ? 0.f : ex2(*cluster.map_shared_rank(&um[r], k) - ref) / total * vunit;
  }
  __syncthreads();
  for (int x = split * blockDim.x + threadIdx.x; x < rows * (HD / 4); x += p.splits * blockDim.x) {
    const int r = x / (HD / 4), c = x % (HD / 4) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < p.splits; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(u0, k) + r * HD + c);
      const float f = share[k][r];
      sum.x += v.x * f; sum.y += v.y * f; sum.z += v.z * f; sum.w += v.w * f;
    }
    store(r, c, sum);
  }
  cluster.sync();                                      // no block leaves while another reads its shared memory
}

inline int allow_smem(unsigned long long& done, const void* kernel, int bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < 64 && (done >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);      // clusters of 16
    if (e == cudaSuccess && dev < 64) done |= 1ull << dev;
  }
  return (int)e;
}

template <typename T, int HD, int NT, bool NARROW>
int run_mma(Kv4Attn p, cudaStream_t st) {
  using S = MmaShape<T, HD, NT, NARROW>;
  const auto kernel = attention_kv4_mma_kernel<T, HD, NT, NARROW>;
  static unsigned long long attr = 0;                  // devices on which the kernel has its attributes
  if (const int e = allow_smem(attr, (const void*)kernel, MOST_WARPS * S::SMEM_WARP)) return e;
  const long long tiles = ceil_div_ll((long long)p.n * p.group, S::ROWS), units = tiles * p.d.heads * p.d.slots;
  if (units * MOST_WARPS * 16 > 0x7fffffffLL) return LLMB_ERR_BAD_ARG;
  // How many warps share a unit.  Units that fill the chip get one warp each, or two where a second round would be a short one (256 x 16
  // heads of 64, up to 1024 tokens: 60 us with one, 54 with two, 56 with four, 68 with eight; 1024 x 16, up to 512: 106, 112, 130, 184); fewer
  // get up to eight, as long as all warps fit on the chip at once (32 x 12, up to 777 tokens: 15.5, 12.8, 11.4, 9.1; 64 x 12: 26, 23, 17, 18), and
  // then a cluster of blocks (4 x 8 heads of 128, 32001 tokens: 142 us in one block, 76, 58, 35, 49 in 2, 4, 8, 16).  The first doubling costs what
  // joining over distributed memory does, about 1 us, and pays from two tiles a warp on; the next ones from one tile a warp on (1 x 12: 1000 tokens
  // 5.6 in one block, 6.5 in two, 1500 6.8 and 7.5; 2000 8.1, 7.7, 6.5 in 1, 2, 4; 4000 10.3 in two, 7.7 in four; heads of 128, 1 x 8, 3000 tokens: 12.3, 8.9,
  // 7.9 in 2, 4, 8).
  const long long fit = (long long)sm_count() * S::WARPS_SM;
  const int most = ceil_div(p.d.capacity, S::TK);
  int log_w = units > fit && units <= 2 * fit && most > 1 ? 1 : 0;
  while (log_w < 3 && (units << (log_w + 1)) <= fit && (2 << log_w) <= most) ++log_w;
  p.splits = 1;
  if (log_w == 3) while (p.splits < MOST_SPLITS && units * 16 * p.splits <= fit && (p.splits == 1 ? 32 : p.splits * 16) <= most) p.splits *= 2;
  const int warps = log_w == 3 ? 8 : 4;
  return launch_pdl_cluster(dim3(p.splits), kernel, dim3((unsigned)(ceil_div_ll(units << log_w, warps) * p.splits)), warps * 32, warps * S::SMEM_WARP, st, p, log_w, (int)tiles);
}
// The tcgen05 kernel takes calls of PROMPT_ROWS rows of a key head and more, if its items (a tile of 128 rows, or two where there are more tiles
// than SMs, of one slot and key head) occupy three fifths of the SMs or the cache is short.  It does not share an item's keys between blocks; the
// kernel above does, and is the faster one where few items have many keys: 64 rows of 1 x 12 heads behind 1000, 8000 and 30000 tokens 20, 109, 390 us
// there and 15, 22, 51 here, one token of 64 heads over one with 30000 tokens 384 and 25; 128 rows of 8 x 16 behind 4000 63 there and 94 here.
// Short caches (up to PROMPT_SHORT tokens) take 7.2 us there and 10.9 here (1 x 12, 64 rows), 500 tokens of 64 heads over one 11.8 and 9.7.
// In 551 calls of 64 to 1024 rows the rule is 1.6 % from the faster kernel's time; what it misses are tiles of 64 to 96 rows on a full chip
// (16 x 12, 64 rows behind 700 tokens: 32 there and 26 here).
constexpr int PROMPT_ROWS = 64, PROMPT_SHORT = 384;
template <typename T, int HD>
int run(const Kv4Attn& p, cudaStream_t st) {
  const long long rows = (long long)p.n * p.group;
  if (sizeof(T) == 2 && HD == 64 && rows >= PROMPT_ROWS) {
    const long long units = (long long)p.d.slots * p.d.heads, tiles = ceil_div_ll(rows, 128);
    const long long items = units * (tiles * units <= sm_count() ? tiles : ceil_div_ll(tiles, 2));
    if (items * 5 >= sm_count() * 3LL || p.d.capacity <= PROMPT_SHORT) return kv4_attention_prompt(p, st);
  }
  constexpr int R8 = sizeof(T) == 4 ? 4 : 8, MOST = HD <= 64 ? 4 : 2;
  if (rows <= R8 / 2) return run_mma<T, HD, 1, true>(p, st);
  if (rows <= R8) return run_mma<T, HD, 1, false>(p, st);
  if (rows <= 2 * R8 || MOST == 2) return run_mma<T, HD, 2, false>(p, st);
  return run_mma<T, HD, MOST, false>(p, st);
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
            a->qb, a->qt, a->qh, a->ob, a->ot, a->oh, a->status, false, false};
  const int elt = a->dtype == LLMB_BF16 ? 2 : 4;
  p.o_vec = ((reinterpret_cast<uintptr_t>(a->out) | (uintptr_t)(a->ob * elt) | (uintptr_t)(a->ot * elt) | (uintptr_t)(a->oh * elt)) & (4 * elt - 1)) == 0;
  p.q_vec = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(a->qb * elt) | (uintptr_t)(a->qt * elt) | (uintptr_t)(a->qh * elt)) & 15) == 0;
  return a->dtype == LLMB_BF16 ? run_type<__nv_bfloat16>(p, st) : run_type<float>(p, st);
}
