// Attention of many new tokens (a prompt) over the 4-bit key/value cache: tcgen05 + TMEM, bf16, heads of 64.
//
// The kernel is built like the causal forward kernel of attention_fwd.cu: a persistent CTA takes pairs of 128-row query tiles that share one stream
// of 128-key blocks; two softmax warpgroups (one thread per row), an output warpgroup, two issuing warps; scores and P in tensor
// memory, O rescaled lazily.  What differs:
//   - a row is (new token, query head of the key head's group); rows see the keys up to their own token's position, from the device's lengths;
//   - no TMA: warps 12 and 15 read the codes and scales of a block's keys and values (from whichever slot keeps the page), turn them into f16
//     and write the swizzled tiles that the tensor core reads (code x scale is exact in f16: cvt and a multiplication for two values);
//   - the output warpgroup brings the next item's rows of q into f16's range by a power of two each (exact) and writes their tiles;
//   - P is f16, up to 2^15: the maximum lags by up to 2^8, the rest of the range goes to small weights.  A weight is off by up to 2^-11 of itself, an
//     eighth of what a bf16 result's own rounding is, or, below f16's normal numbers, by 2^-32 of their sum.
// 16 x 12 heads, ragged prompts of up to 1000 tokens: 72 us; the kernel for few rows (mma.sync, 32 rows a warp) takes 158 us there.  All prompts
// 1024 long: 90 us, the causal forward kernel on bf16 keys 69.  A softmax warp's chain (scores, maximum, 2^x, P) per block bounds both; the conversion
// of the codes adds 6 us.
#include "kv4.cuh"
#include "attention_common.cuh"
using namespace kv4;

namespace {
constexpr int KP_NS = 3;                                  // K/V ring depth (32 KB per stage)
constexpr int KP_RAW = 3, RAW_BYTES = 128 * 36;           // blocks of codes and scales on their way, per operand
constexpr int KP_THREADS = 512;
constexpr int KP_SORT = 256;                               // most pairs of a slot and a pair of tiles that are sorted by their cost
constexpr int KP_SMEM = 4 * T128 /*Q: 2 buffers x 2 tiles*/ + KP_NS * 2 * T128 /*K,V ring*/ + 2 * KP_RAW * RAW_BYTES /*codes and scales*/ + 1024 /*alignment*/ + 512 /*barriers*/ +
                        2048 /*row sums*/ + 2048 /*row factors*/ + KP_SORT * 20 /*slots and pairs of tiles by cost*/;
constexpr uint32_t IDESC_QK = make_idesc(FMT_F16, FMT_F16, 0, 0, 128, 128);
constexpr uint32_t IDESC_PV = make_idesc(FMT_F16, FMT_F16, 0, 1, 128, 64);     // A (P) K-major from TMEM, B (V) stored [keys, HS]
constexpr float P_SHIFT = 7.f;                            // P <= 2^(7 + 8)

#define KP_FAIL() do { atomicExch(p.status, LLMB_ERR_TIMEOUT); failed = true; } while (0)

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) { uint32_t d; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo)); return d; }
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) { uint32_t d; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}

// A work item: one (slot, key head) and the query tiles t0, t0 + 1 (tpi 2; or t0 alone).  nb: key blocks that the tile sees, 0 where it has no
// rows or sees nothing; the second tile sees no fewer than the first unless it has no rows.
//
// Items are dealt out by decreasing cost, forwards and backwards in turns.  What a slot's tiles cost is known on the device alone: where there are
// no more than KP_SORT pairs of a slot and a pair of tiles, every CTA sorts those by the blocks that they see (16 ragged prompts of up to 1000
// tokens: at most 27 blocks on a CTA, 24.9 on average; 31 by the pairs alone).  Else the last pairs of all slots come first.
struct KpItem { int s, h, t0, len, cnt, rows[2], nb[2], most; bool valid; };
struct KpGrid { int n_pairs, tpi, sorted; };
struct KpEntry { int s, pair, len, cnt; };
__device__ __forceinline__ int kp_token(const Kv4Attn& p, int row) { return p.group == 1 ? row : row / p.group; }
__device__ __forceinline__ KpEntry kp_entry(const Kv4Attn& p, int s, int pair) {
  return KpEntry{s, pair, min(max(p.lens[s], 0), p.d.capacity), p.counts ? min(max(p.counts[s], 0), p.n) : p.n};
}
__device__ __forceinline__ KpItem kp_of(const Kv4Attn& p, const KpGrid& g, const KpEntry& e, int h) {
  KpItem it;
  it.valid = true;
  it.s = e.s; it.h = h; it.t0 = g.tpi * e.pair; it.len = e.len; it.cnt = e.cnt;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = (it.t0 + t) * TILE;
    it.rows[t] = t < g.tpi ? max(0, min(TILE, it.cnt * p.group - first)) : 0;
    it.nb[t] = it.rows[t] ? ceil_div(max(0, it.len - it.cnt + kp_token(p, first + it.rows[t] - 1) + 1), TILE) : 0;
  }
  it.most = max(it.nb[0], it.nb[1]);
  return it;
}
// item k of this CTA
__device__ __forceinline__ KpItem kp_item(const Kv4Attn& p, const KpGrid& g, const KpEntry* order, int k) {
  const long long index = (long long)k * gridDim.x + (k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  const int entries = p.d.slots * g.n_pairs;              // times heads below 2^31 (host)
  if (index >= (long long)entries * p.d.heads) { KpItem none; none.valid = false; none.most = 0; return none; }
  const int entry = (int)index / p.d.heads, h = (int)index - entry * p.d.heads;
  if (g.sorted) return kp_of(p, g, order[entry], h);
  const int back = entry / p.d.slots;
  return kp_of(p, g, kp_entry(p, entry - back * p.d.slots, g.n_pairs - 1 - back), h);
}

__global__ void __launch_bounds__(KP_THREADS, 1) attention_kv4_prompt_kernel(const Kv4Attn p, const KpGrid grid, const int o_vec) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = sm;                                 // buffer qb: tile t0 at qb*2*T128, tile t0+1 at +T128
  unsigned char* sKV = sQ + 4 * T128;                     // stage s: K block at s*2*T128, V block at +T128
  unsigned char* sRaw = sKV + KP_NS * 2 * T128;           // keys' blocks, then values': codes of 128 tokens, then scales
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + 2 * KP_RAW * RAW_BYTES);
  uint64_t* q_full = bars;                                // [2] the output warpgroup's four warps
  uint64_t* q_empty = q_full + 2;                         // [lane][2] the lane's last score product of the item is complete
  uint64_t* kv_full = q_empty + 4;                        // [NS] the two warps that write K and V
  uint64_t* kv_empty = kv_full + KP_NS;                   // [lane][NS] the lane is done with the stage
  uint64_t* s_full = kv_empty + 2 * KP_NS;                // [2] per lane: S is in TMEM
  uint64_t* s_free = s_full + 2;                          // [2] per lane: the softmax warps hold S in registers
  uint64_t* p_full = s_free + 2;                          // [2] per lane: P is in TMEM (and O rescaled if needed)
  uint64_t* pv_done = p_full + 2;                         // [2] per lane: O += P V complete (P may be overwritten)
  uint64_t* o_free = pv_done + 2;                         // [2] per lane: the item's output has left TMEM
  uint64_t* fin = o_free + 2;                             // [2] per lane: the item's row statistics are in shared memory
  uint64_t* raw_full = fin + 2;                           // [2][RAW] a block's codes and scales are in shared memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_full + 2 * KP_RAW);
  float* stats = reinterpret_cast<float*>(bars + 64);     // [lane][item parity][l][128 rows] (m is not needed)
  float* factor = stats + 512;                            // [qb][tile][128 rows]: products to log2 units
  KpEntry* order = reinterpret_cast<KpEntry*>(factor + 512);               // by decreasing cost
  int* cost = reinterpret_cast<int*>(order + KP_SORT);

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4); mbar_init(&q_empty[i], 1); mbar_init(&q_empty[2 + i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 4); mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1); mbar_init(&o_free[i], 4); mbar_init(&fin[i], 4);
    }
    for (int i = 0; i < 2 * KP_RAW; ++i) mbar_init(&raw_full[i], 1);
    for (int i = 0; i < KP_NS; ++i) { mbar_init(&kv_full[i], 2); mbar_init(&kv_empty[i], 1); mbar_init(&kv_empty[KP_NS + i], 1); }
    fence_barrier_init();
  }
  if (warp == 13) tmem_alloc<512>(tmem_slot);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool failed = false;
  pdl_trigger();
  pdl_wait();
  if (grid.sorted) {
    const int entries = p.d.slots * grid.n_pairs;         // at most KP_SORT < KP_THREADS
    KpEntry mine{};
    if (tid < entries) {
      const int pair = tid / p.d.slots;
      mine = kp_entry(p, tid - pair * p.d.slots, pair);
      const KpItem it = kp_of(p, grid, mine, 0);
      cost[tid] = it.rows[0] ? it.most + 1 : 0;
    }
    __syncthreads();
    if (tid < entries) {
      int rank = 0;
      for (int o = 0; o < entries; ++o) rank += cost[o] > cost[tid] || (cost[o] == cost[tid] && o < tid);
      order[rank] = mine;
    }
    __syncthreads();
  }
  // Registers: 2 x 128 x 176 + 2 x 128 x 80 = 65536 = the 512 x 128 that the CTA was launched with; each role sets its limit in its own branch.
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 12 || warp == 15) {
      // ---------------------------------------------------------- keys (warp 12) and values (warp 15) into the ring
      // Untiled bulk copies bring a block's codes and scales (contiguous within a page) into a ring of the warp's own, three blocks ahead of their
      // conversion; held in registers instead, they were spilled, and every block waited for its loads (145 us for the prompts above).
      const bool is_v = warp == 15;
      const uint8_t* codes = (is_v ? p.d.vc : p.d.kc) + p.layer * p.d.code_layer;
      const uint8_t* scales = (is_v ? p.d.vs : p.d.ks) + p.layer * p.d.scale_layer;
      unsigned char* raw = sRaw + (is_v ? KP_RAW * RAW_BYTES : 0);
      uint64_t* full = raw_full + (is_v ? KP_RAW : 0);
      const int half = lane & 1, key0 = lane >> 1;        // a lane takes half a row, 16 bytes of codes, of the rows key0 + 16 x
      KpItem it = kp_item(p, grid, order, 0);
      int k = 0, j = 0, issued = 0;
      uint32_t state = 0;                                 // four bits per stage: page 0 / 1 names no slot, page 1 lies behind the cache
      auto issue = [&]() {
        while (it.valid && j >= it.most) { j = 0; it = kp_item(p, grid, order, ++k); }
        if (!it.valid) return;
        const int st = issued % KP_RAW, page0 = 2 * j, pages = p.d.capacity / PAGE;
        const bool two = page0 + 1 < pages;
        int s0 = it.s, s1 = it.s;
        if (p.pages) {
          s0 = p.pages[(long long)it.s * pages + page0];
          if (two) s1 = p.pages[(long long)it.s * pages + page0 + 1];
        }
        const bool b0 = s0 < 0 || s0 >= p.d.slots, b1 = s1 < 0 || s1 >= p.d.slots;
        if (b0) s0 = it.s;
        if (b1) s1 = it.s;
        state = (state & ~(15u << (4 * st))) | (uint32_t)(b0 | b1 << 1 | !two << 2) << (4 * st);
        if (lane == 0) {
          const long long at = (long long)it.h * pages + page0;
          unsigned char* dst = raw + st * RAW_BYTES;
          mbar_expect_tx(&full[st], two ? RAW_BYTES : RAW_BYTES / 2);
          bulk_load_1d(dst, codes + s0 * p.d.code_slot + at * PAGE * 32, PAGE * 32, &full[st]);
          bulk_load_1d(dst + 2 * PAGE * 32, scales + s0 * p.d.scale_slot + at * PAGE * 4, PAGE * 4, &full[st]);
          if (two) {
            bulk_load_1d(dst + PAGE * 32, codes + s1 * p.d.code_slot + (at + 1) * PAGE * 32, PAGE * 32, &full[st]);
            bulk_load_1d(dst + 2 * PAGE * 32 + PAGE * 4, scales + s1 * p.d.scale_slot + (at + 1) * PAGE * 4, PAGE * 4, &full[st]);
          }
        }
        ++j; ++issued;
      };
      for (int x = 0; x < KP_RAW; ++x) issue();
      for (int g = 0; g < issued && !failed; ++g) {
        const int st = g % KP_NS, rs = g % KP_RAW;
        if (!mbar_wait(&full[rs], (g / KP_RAW) & 1)) { KP_FAIL(); break; }
        if (g >= KP_NS && !(mbar_wait(&kv_empty[st], ((g / KP_NS) + 1) & 1) && mbar_wait(&kv_empty[KP_NS + st], ((g / KP_NS) + 1) & 1))) { KP_FAIL(); break; }
        unsigned char* tile = sKV + st * 2 * T128 + (is_v ? T128 : 0);
        const unsigned char* src = raw + rs * RAW_BYTES;
        const uint32_t how = state >> (4 * rs);
#pragma unroll 4
        for (int x = 0; x < 8; ++x) {
          const int row = key0 + 16 * x;
          const uint4 w = *reinterpret_cast<const uint4*>(src + row * 32 + half * 16);
          uint32_t f = *reinterpret_cast<const uint16_t*>(src + 2 * PAGE * 32 + row * 4 + half * 2);
          if (x >= 4 && (how & 4)) f = 0;                 // behind the cache: whatever lies there, times 0
          if (how & (x < 4 ? 1 : 2)) f = 0x7f7f;          // NaN for whoever sees the page
          uint32_t two = e4m3x2_f16x2(f);
          // A NaN scale of a value becomes 448: the key's scales are NaN as well and say so to the rows that see it, and to no other.
          if (is_v) asm("min.f16x2 %0, %0, %1;" : "+r"(two) : "r"(0x5f005f00u));
          const uint32_t s0 = __byte_perm(two, two, 0x1010), s1 = __byte_perm(two, two, 0x3232);
          const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t h[4];
            unpack8(word[y], h);
#pragma unroll
            for (int z = 0; z < 4; ++z) h[z] = mul2(h[z], y < 2 ? s0 : s1);
            *reinterpret_cast<uint4*>(tile + sw128(row, half * 4 + y)) = make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
        fence_proxy_async();
        __syncwarp();                                     // every lane has read the raw stage, too
        if (lane == 0) mbar_arrive(&kv_full[st]);
        issue();
      }
      if (failed)                                         // leave with no copy in flight
        for (int x = max(0, issued - KP_RAW); x < issued; ++x) mbar_wait(&full[x % KP_RAW], (x / KP_RAW) & 1);
    } else {
      // ---------------------------------------------------------- MMA issuer of lane r
      const int r = warp - 13;
      const uint32_t tS = tmem + r * 128, tO = tmem + 256 + r * 64, tP = tmem + 384 + r * 64;
      uint64_t* my_q_empty = q_empty + 2 * r;
      uint64_t* my_kv_empty = kv_empty + KP_NS * r;
      int g0 = 0, cs = 0, cp = 0, no = 0;                 // blocks before this item; S / PV / item counts of this lane
      const uint64_t q_desc0 = make_smem_desc(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc0 = make_smem_desc(smem_u32(sKV), 16, 1024);
      const uint64_t v_desc0 = make_smem_desc(smem_u32(sKV + T128), 8192, 1024);
      for (int k = 0; !failed; ++k) {
        const KpItem it = kp_item(p, grid, order, k);
        if (!it.valid) break;
        const int qb = k & 1, tt = r ^ (k & 1), nbt = tt ? it.nb[1] : it.nb[0];
        const uint64_t q_desc = q_desc0 + (uint64_t)(((qb * 2 + tt) * T128) >> 4);
        // the item's Q buffer and every K/V stage are acquired before they are released, also where this lane does not read them
        if (!mbar_wait(&q_full[qb], (k >> 1) & 1)) { KP_FAIL(); break; }
        if (nbt > 0) {
          auto issue_s = [&](int j) {
            const int g = g0 + j, st = g % KP_NS;
            if (!mbar_wait(&kv_full[st], (g / KP_NS) & 1)) { KP_FAIL(); return; }
            if (cs >= 1 && !mbar_wait(&s_free[r], (cs - 1) & 1)) { KP_FAIL(); return; }
            fence_after_sync();
            const uint64_t k_desc = k_desc0 + (uint64_t)((st * 2 * T128) >> 4);
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < HS / 16; ++ks)                                              // S = Q K^T
                umma_ss<KIND_F16>(tS, q_desc + 2 * ks, k_desc + 2 * ks, IDESC_QK, ks > 0 ? 1u : 0u);
              umma_commit(&s_full[r]);
              if (j == nbt - 1) umma_commit(&my_q_empty[qb]);
            }
            __syncwarp();
            ++cs;
          };
          issue_s(0);
          for (int j = 0; j < nbt && !failed; ++j) {
            if (j + 1 < nbt) issue_s(j + 1);
            if (failed) break;
            const int st = (g0 + j) % KP_NS;
            if (!mbar_wait(&p_full[r], cp & 1)) { KP_FAIL(); break; }
            if (j == 0 && no >= 1 && !mbar_wait(&o_free[r], (no - 1) & 1)) { KP_FAIL(); break; }
            fence_after_sync();
            const uint64_t vd = v_desc0 + (uint64_t)((st * 2 * T128) >> 4);
            const uint32_t acc0 = j > 0 ? 1u : 0u;
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < TILE / 16; ++ks)                                            // O (+)= P V
                umma_ts(tO, tP + ks * 8, vd + 128 * ks, IDESC_PV, ks > 0 ? 1u : acc0);
              umma_commit(&pv_done[r]);
              umma_commit(&my_kv_empty[st]);
            }
            __syncwarp();
            ++cp;
          }
          ++no;
        } else if (elect_one()) {
          umma_commit(&my_q_empty[qb]);                   // nothing of this lane reads the Q buffer
        }
        if (failed) break;
        // blocks this lane does not look at: release them in order behind the lane's own products
        for (int j = nbt; j < it.most && !failed; ++j) {
          const int g = g0 + j, st = g % KP_NS;
          if (!mbar_wait(&kv_full[st], (g / KP_NS) & 1)) { KP_FAIL(); break; }
          if (elect_one()) umma_commit(&my_kv_empty[st]);
          __syncwarp();
        }
        g0 += it.most;
      }
    }
  } else if (warp >= 8) {
    // -------------------------------------------------------------- rows of q in, rows of the output out: one thread per row
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const float vunit = pow2(p.d.v_exp);
    int cp[2] = {0, 0}, ni[2] = {0, 0};                   // per lane: products / items so far
    auto load_q = [&](int k) {
      const KpItem it = kp_item(p, grid, order, k);
      if (!it.valid) return;
      const int qb = k & 1;
      if (k >= 2 && !(mbar_wait(&q_empty[qb], ((k >> 1) + 1) & 1) && mbar_wait(&q_empty[2 + qb], ((k >> 1) + 1) & 1))) { KP_FAIL(); return; }
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        uint32_t x[32];
#pragma unroll
        for (int y = 0; y < 32; ++y) x[y] = 0;
        if (row < (t ? it.rows[1] : it.rows[0])) {
          const int at = (it.t0 + t) * TILE + row, token = kp_token(p, at);
          const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q) + (it.s * p.qb + token * p.qt + (it.h * p.group + at - token * p.group) * p.qh);
          if (p.q_vec) {
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const uint4 v = *reinterpret_cast<const uint4*>(q + y * 8);
              x[4 * y] = v.x; x[4 * y + 1] = v.y; x[4 * y + 2] = v.z; x[4 * y + 3] = v.w;
            }
          } else {
            const unsigned short* u = reinterpret_cast<const unsigned short*>(q);
#pragma unroll
            for (int y = 0; y < 32; ++y) x[y] = u[2 * y] | (uint32_t)u[2 * y + 1] << 16;
          }
        }
        uint32_t m2 = x[0] & 0x7fff7fffu;                 // of magnitudes, as unsigned numbers: NaN and infinity come out on top
#pragma unroll
        for (int y = 1; y < 32; ++y) m2 = __vmaxu2(m2, x[y] & 0x7fff7fffu);
        const uint32_t top = max(m2 & 0xffffu, m2 >> 16);
        // the largest value lies in [2^14, 2^15) after the shift; a row without one of 2^-86 or more has no score of any size
        const int e = max((int)(top >> 7) - 141, -100);
        const float down = top < 0x7f80u ? (p.scale_log2 < 0.f ? -1.f : p.scale_log2 == 0.f ? 0.f : 1.f) * pow2(-e) : __int_as_float(0x7fc00000);
        unsigned char* tile = sQ + (qb * 2 + t) * T128;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          uint32_t h[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) h[z] = f16x2(__uint_as_float(x[4 * y + z] << 16) * down, __uint_as_float(x[4 * y + z] & 0xffff0000u) * down);
          *reinterpret_cast<uint4*>(tile + sw128(row, y)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        factor[(qb * 2 + t) * 128 + row] = p.scale_log2 == 0.f ? 1.f : fmaxf(fabsf(p.scale_log2) * pow2(e / 2) * pow2(e - e / 2) * pow2(p.d.k_exp), 1e-37f);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[qb]);
    };
    load_q(0);
    for (int k = 0; !failed; ++k) {
      const KpItem it = kp_item(p, grid, order, k);
      if (!it.valid) break;
      load_q(k + 1);
      if (failed) break;
#pragma unroll 1
      for (int tt = 0; tt < 2 && !failed; ++tt) {
        const int r = tt ^ (k & 1), nbt = tt ? it.nb[1] : it.nb[0], rows = tt ? it.rows[1] : it.rows[0];
        const int at = (it.t0 + tt) * TILE + row, token = kp_token(p, at);
        __nv_bfloat16* o_row = reinterpret_cast<__nv_bfloat16*>(p.out) + (it.s * p.ob + token * p.ot + (it.h * p.group + at - token * p.group) * p.oh);
        auto store8 = [&](int c, const uint4 v) {
          if (o_vec) *reinterpret_cast<uint4*>(o_row + c) = v;
          else {
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int z = 0; z < 8; ++z) reinterpret_cast<unsigned short*>(o_row)[c + z] = (unsigned short)(u[z / 2] >> (16 * (z & 1)));
          }
        };
        if (nbt == 0) {                                   // rows that see nothing
          if (row < rows)
#pragma unroll
            for (int c = 0; c < 64; c += 8) store8(c, make_uint4(0, 0, 0, 0));
          continue;
        }
        if (!mbar_wait(&fin[r], ni[r] & 1)) { KP_FAIL(); break; }
        cp[r] += nbt;
        const float l_run = stats[(r * 2 + (ni[r] & 1)) * 128 + row];
        ++ni[r];
        if (!mbar_wait(&pv_done[r], (cp[r] - 1) & 1)) { KP_FAIL(); break; }      // the tile's last product
        fence_after_sync();
        const uint32_t tO = tmem + 256 + r * 64 + lane_addr;
        const float inv = l_run == 0.f ? 0.f : vunit / l_run;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t o[32];
          tmem_ld32(tO + half * 32, o);
          tmem_wait_ld();
          if (half == 1) {                                // O has left TMEM: the lane's next item may overwrite it
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[r]);
          }
          if (row < rows) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t u[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) u[z] = pack_bf16x2(__uint_as_float(o[8 * c + 2 * z]) * inv, __uint_as_float(o[8 * c + 2 * z + 1]) * inv);
              store8(half * 32 + c * 8, make_uint4(u[0], u[1], u[2], u[3]));
            }
          }
        }
      }
    }
  } else {
    // -------------------------------------------------------------- softmax warps of lane r: one thread per query row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int r = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + r * 128 + lane_addr, tO = tmem + 256 + r * 64 + lane_addr, tP = tmem + 384 + r * 64 + lane_addr;
    int cs = 0, cp = 0, ni = 0;
    for (int k = 0; !failed; ++k) {
      const KpItem it = kp_item(p, grid, order, k);
      if (!it.valid) break;
      const int tt = r ^ (k & 1), nbt = tt ? it.nb[1] : it.nb[0];
      if (nbt == 0) continue;
      // keys that the row sees; a row that is none sees what the last one does
      const int see = it.len - it.cnt + kp_token(p, (it.t0 + tt) * TILE + min(row, (tt ? it.rows[1] : it.rows[0]) - 1)) + 1;
      float m_run = -INFINITY, l_run = 0.f, sc = 1.f;     // m_run in log2 units
      for (int j = 0; j < nbt; ++j) {
        if (!mbar_wait(&s_full[r], cs & 1)) { KP_FAIL(); break; }
        fence_after_sync();
        if (j == 0) sc = factor[((k & 1) * 2 + tt) * 128 + row];
        uint32_t s[128];
        {
          uint32_t (&q0)[32] = *reinterpret_cast<uint32_t (*)[32]>(&s[0]);
          uint32_t (&q1)[32] = *reinterpret_cast<uint32_t (*)[32]>(&s[32]);
          uint32_t (&q2)[32] = *reinterpret_cast<uint32_t (*)[32]>(&s[64]);
          uint32_t (&q3)[32] = *reinterpret_cast<uint32_t (*)[32]>(&s[96]);
          tmem_ld32(tS, q0); tmem_ld32(tS + 32, q1); tmem_ld32(tS + 64, q2); tmem_ld32(tS + 96, q3);
        }
        tmem_wait_ld();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[r]);           // the next block's scores may overwrite S now
        ++cs;
        const int lim = see - j * TILE;
#pragma unroll
        for (int c = 0; c < 4; ++c) {                     // keys behind the row's token
          if (__any_sync(0xffffffffu, lim < 32 * (c + 1))) {
#pragma unroll
            for (int x = 32 * c; x < 32 * (c + 1); ++x)
              if (x >= lim) s[x] = 0xff800000u;
          }
        }
        float mx4[4];                                     // four independent chains: the row maximum is latency, not work
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx4[c] = fmaxf(__uint_as_float(s[c * 32]), __uint_as_float(s[c * 32 + 1]));
#pragma unroll
          for (int x = 2; x < 32; x += 2) mx4[c] = max3(mx4[c], __uint_as_float(s[c * 32 + x]), __uint_as_float(s[c * 32 + x + 1]));
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
        // the reference maximum only moves when it grew by more than 8 (a factor 256 in p): rescales of O become rare
        float m_new = fmaxf(m_run, mx);
        if (m_new - m_run <= 8.0f) m_new = m_run;
        const float ref = m_new == -INFINITY ? 0.f : m_new;       // a row that has seen nothing yet
        const float alpha = ex2_approx(m_run - ref);
        m_run = m_new;
        // O += P(j-1) V must be complete before O is rescaled and before P is overwritten
        if (cp >= 1 && !mbar_wait(&pv_done[r], (cp - 1) & 1)) { KP_FAIL(); break; }
        fence_after_sync();
        if (j > 0 && !__all_sync(0xffffffffu, alpha == 1.0f)) {
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            uint32_t o[32];
            tmem_ld32(tO + half * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
            tmem_st32(tO + half * 32, o);
          }
        }
        const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(P_SHIFT - ref, P_SHIFT - ref);
        float2 acc[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int x = 0; x < 64; ++x) {
          const float2 t2 = __ffma2_rn(make_float2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1])), sc2, nm2);
          const float e0 = ex2_approx(t2.x), e1 = ex2_approx(t2.y);
          acc[x & 3] = __fadd2_rn(acc[x & 3], make_float2(e0, e1));
          s[x] = f16x2(e0, e1);                           // P(j) as f16 pairs replaces the scores already consumed
        }
        {
          const uint32_t (&p0)[32] = *reinterpret_cast<const uint32_t (*)[32]>(&s[0]);
          const uint32_t (&p1)[32] = *reinterpret_cast<const uint32_t (*)[32]>(&s[32]);
          tmem_st32(tP, p0); tmem_st32(tP + 32, p1);
        }
        const float2 a01 = __fadd2_rn(acc[0], acc[1]), a23 = __fadd2_rn(acc[2], acc[3]);
        l_run = l_run * alpha + ((a01.x + a01.y) + (a23.x + a23.y));
        tmem_wait_st();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[r]);
        ++cp;
      }
      if (failed) break;
      // Hand the row sums to the output warpgroup and go on with the next item.  The previous item's output must have been taken first,
      // so that `fin` never runs two phases ahead of its reader.
      if (ni >= 1 && !mbar_wait(&o_free[r], (ni - 1) & 1)) { KP_FAIL(); break; }
      stats[(r * 2 + (ni & 1)) * 128 + row] = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(&fin[r]);
      ++ni;
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 13) { fence_after_sync(); tmem_dealloc<512>(tmem); }
}
}  // namespace

int kv4_attention_prompt(const Kv4Attn& p, cudaStream_t st) {
  static unsigned long long attr = 0;                     // devices on which the kernel may take its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < 64 && (attr >> dev & 1))) {
    e = cudaFuncSetAttribute(attention_kv4_prompt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KP_SMEM);
    if (e == cudaSuccess && dev < 64) attr |= 1ull << dev;
  }
  if (e) return (int)e;
  const long long rows = (long long)p.n * p.group, units = (long long)p.d.slots * p.d.heads;
  KpGrid g{};
  const long long n_t = ceil_div_ll(rows, TILE);
  // pairs of tiles share the key blocks; where the chip has an SM for every tile, a tile alone gets an SM's exponential unit to itself
  g.tpi = n_t * units <= sm_count() ? 1 : 2;
  g.n_pairs = (int)ceil_div_ll(n_t, g.tpi);
  const long long items = g.n_pairs * units;
  if (items > 0x7fffffffLL) return LLMB_ERR_BAD_ARG;
  g.sorted = p.counts != nullptr && (long long)p.d.slots * g.n_pairs <= KP_SORT;
  const int ctas = items < sm_count() ? (int)items : sm_count();
  const bool o_vec = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.ob * 2) | (uintptr_t)(p.ot * 2) | (uintptr_t)(p.oh * 2)) & 15) == 0;
  return launch_pdl(attention_kv4_prompt_kernel, ctas, KP_THREADS, KP_SMEM, st, p, g, (int)o_vec);
}
