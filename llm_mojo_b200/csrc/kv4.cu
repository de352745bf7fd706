// The 4-bit key/value cache (layout: kv4.cuh): rounding new keys and values into it, reading it back, and following a beam search.
//
// This file has no counterpart in the reference project, whose inference runs the whole forward pass for every token
// (infer_gpt2.mojo:56-144).
#include "kv4.cuh"
using namespace llmb;
using namespace kv4;

namespace {
struct RowStrides { long long b, t, h; };            // elements: sequence, token, head; the values of a head lie densely

// Sixteen values from p on as pairs of floats, and the largest magnitude among them: NaN if there is one, infinite if that is.
// VEC: 16-byte loads.
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) { uint32_t d; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
__device__ __forceinline__ float max_nan(float a, float b) { float d; asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }
template <bool VEC> __device__ __forceinline__ void load16(uint32_t (&w)[8], const __nv_bfloat16* p) {
  if (VEC) {
    const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 8);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = u[2 * j] | (uint32_t)u[2 * j + 1] << 16;
  }
}
template <bool VEC> __device__ __forceinline__ void load16(uint32_t (&w)[16], const float* p) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (VEC) { const uint4 a = *reinterpret_cast<const uint4*>(p + 4 * j); w[4 * j] = a.x; w[4 * j + 1] = a.y; w[4 * j + 2] = a.z; w[4 * j + 3] = a.w; }
    else {
#pragma unroll
      for (int z = 0; z < 4; ++z) w[4 * j + z] = __float_as_uint(p[4 * j + z]);
    }
  }
}
__device__ __forceinline__ float amax16(const uint32_t (&w)[8]) {
  uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int j = 1; j < 8; ++j) m = max_nan_bf16x2(m, w[j] & 0x7fff7fffu);
  return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}
__device__ __forceinline__ float amax16(const uint32_t (&w)[16]) {
  float m = fabsf(__uint_as_float(w[0]));
#pragma unroll
  for (int j = 1; j < 16; ++j) m = max_nan(m, fabsf(__uint_as_float(w[j])));
  return m;
}
__device__ __forceinline__ float2 pair(const uint32_t (&w)[8], int j) { return make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u)); }
__device__ __forceinline__ float2 pair(const uint32_t (&w)[16], int j) { return make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1])); }

// r / d for r below the bound under which the host found `mul` = ceil(2^32 / d) exact (r d < 2^32), by a division else
struct Divisor { unsigned d, mul; };
__device__ __forceinline__ unsigned quotient(unsigned r, const Divisor& v) { return v.mul ? __umulhi(r, v.mul) : r / v.d; }

template <int HD> struct AppendGroup { static constexpr int value = HD <= 32 ? 4 : HD <= 64 ? 8 : 16; };

// One thread per block of 16 values; the threads of a row's key blocks and of its value blocks are neighbours in a warp (GROUP of them, some
// idle where HD / 8 is no power of two) because a non-finite value marks all of them.  A block of threads stays with a slot; its rows are counted
// (token, head), the head fastest: the inputs, most of the bytes, are then read as they lie, and what is written meets in L2.
// The codes are those of the exact quotients x / s, s the scale.  A tie between two levels is a product of a midpoint's 3 bits and the scale's 4.
// The correctly rounded quotient is a midpoint only where x / s is one; a product with the rounded reciprocal is not (fl(1 / 0.875) 0.75 x 0.875
// lies above 0.75).  It takes three operations from the correctly rounded reciprocal r (Markstein: q = x r, q + r (x - q s)), on pairs one and
// a half; r takes one Newton step from the approximate one, which is the correctly rounded one for all eight significands that scales have.
// The negative quotient is made (with -r for r) and the codes' signs are turned back: the correction adds a zero to q = x r = -0 and would make
// it +0; to -q it adds one of q's sign, so that zeros keep theirs.
// The ALU pipe is the busiest unit (67 % of its cycles, issue slots 59 %; about 165 instructions for 16 values, idle lanes among them): 16 x 25 heads,
// prompts of 500 to 1000 tokens, 100 MB: 28.7 us in bf16, 35.1 in fp32 (179 MB).
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4Desc d, int layer, const T* __restrict__ k, const T* __restrict__ v,
                                                         const int* __restrict__ start, const int* __restrict__ counts, int n, Divisor by_heads, RowStrides sk, RowStrides sv) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = HD / BLOCK, GROUP = AppendGroup<HD>::value, ROWS = 256 / GROUP, FLIGHT = VEC ? 32 / (int)sizeof(T) / 8 : 1;
  const int lane = threadIdx.x % 32, at = threadIdx.x % GROUP;
  const unsigned group = ((1u << GROUP) - 1) << (lane - at);
  const bool is_v = at >= NB;
  const int blk = is_v ? at - NB : at;
  const RowStrides st = is_v ? sv : sk;
  const int e = is_v ? d.v_exp : d.k_exp;
  const float unit = pow2(e), per_unit = pow2(-e);
  for (int s = blockIdx.y; s < d.slots; s += gridDim.y) {
    const long long first = start[s];
    const int cnt = counts ? min(counts[s], n) : n;
    // tokens lo .. hi - 1 have a place in the cache
    const int lo = first < 0 ? (int)min(-first, (long long)n) : 0, hi = (int)max(min((long long)cnt, d.capacity - first), 0LL);
    const unsigned rows = (unsigned)d.heads * n;       // below 2^31 (host)
    const T* const from = (is_v ? v : k) + s * st.b + blk * BLOCK;
    uint8_t* const codes = (is_v ? d.vc : d.kc) + layer * d.code_layer + s * d.code_slot + first * (HD / 2) + blk * 8;
    uint8_t* const scales = (is_v ? d.vs : d.ks) + layer * d.scale_layer + s * d.scale_slot + first * NB + blk;
    // whole groups walk the rows together, so that the votes below have all their lanes
    for (unsigned r0 = blockIdx.x * (ROWS * FLIGHT); r0 < rows; r0 += gridDim.x * (ROWS * FLIGHT)) {
      uint32_t w[FLIGHT][4 * sizeof(T)];
      int token[FLIGHT], head[FLIGHT];
      bool live[FLIGHT];
#pragma unroll
      for (int y = 0; y < FLIGHT; ++y) {
        const unsigned r = r0 + y * ROWS + threadIdx.x / GROUP, i = quotient(r, by_heads);
        token[y] = i; head[y] = r - i * by_heads.d;
        live[y] = r < rows && at < 2 * NB && token[y] >= lo && token[y] < hi;
#pragma unroll
        for (int j = 0; j < 4 * (int)sizeof(T); ++j) w[y][j] = 0;
        if (live[y]) load16<VEC>(w[y], from + token[y] * st.t + head[y] * st.h);
      }
#pragma unroll
      for (int y = 0; y < FLIGHT; ++y) {
        const float amax = amax16(w[y]);
        const bool bad = (__ballot_sync(0xffffffffu, !(amax <= 3.402823466e38f)) & group) != 0;
        if (!live[y]) continue;
        const float a = fminf(amax * per_unit, 1e30f), sixth = 1.f / 6.f, q6 = a * sixth;
        const uint32_t sc = e4m3(fmaf(fmaf(-q6, 6.f, a), sixth, q6));
        const float s32 = e4m3_f32(sc) * unit;
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s32));
        r = fmaf(fmaf(-s32, r, 1.f), r, r);
        const float2 r2 = make_float2(-r, -r), s2 = make_float2(s32, s32);
        uint32_t code[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float2 x = pair(w[y], j);
          if (sc == 0x7e) { x.x = fminf(fmaxf(x.x, -8.f * s32), 8.f * s32); x.y = fminf(fmaxf(x.y, -8.f * s32), 8.f * s32); }      // what saturates stays in range
          const float2 q = __fmul2_rn(x, r2), t = __ffma2_rn(__ffma2_rn(q, s2, x), r2, q);      // -x / s
          code[j] = e2m1x2(t.x, t.y);
        }
        uint2 c;
        c.x = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
        c.y = __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410);
        c.x ^= 0x88888888u; c.y ^= 0x88888888u;        // of x / s
        if (bad || sc == 0) c = make_uint2(0, 0);
        const long long row = (long long)head[y] * d.capacity + token[y];
        *reinterpret_cast<uint2*>(codes + row * (HD / 2)) = c;
        scales[row * NB] = bad ? 0x7f : (uint8_t)sc;
      }
    }
  }
}

// One thread per 16 bytes of an output, of both the key and the value; the pieces of a row, then its heads, then its tokens are neighbours: the
// stores, which are most of the bytes, are dense where the outputs are.  A block stays with one slot of one layer.  Stores bound it: 24 layers
// of 64 slots, 64 tokens of 16 heads of 64 (403 MB written, 113 MB read) take 100 us;
// a plain fill runs at 3.94 TB/s, 102 us for as much.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(256) kv4_values_kernel(const Kv4Desc d, int layer, T* __restrict__ ko, T* __restrict__ vo, const int* __restrict__ start,
                                                         const int* __restrict__ pages, int n, long long out_layer, RowStrides sk, RowStrides sv) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = HD / BLOCK, N = 16 / sizeof(T), PIECES = HD / N, FLIGHT = 4;
  const unsigned total = (unsigned)n * d.heads * PIECES, planes = (layer < 0 ? d.layers : 1) * d.slots;      // below 2^31 (host)
  for (unsigned plane = blockIdx.y; plane < planes; plane += gridDim.y) {
    const int l = plane / d.slots, s = plane - l * d.slots;
    const long long first = start[s];
    const long long cl = (layer < 0 ? l : layer) * d.code_layer, fl = (layer < 0 ? l : layer) * d.scale_layer;
    for (unsigned x0 = blockIdx.x * (256 * FLIGHT) + threadIdx.x; x0 < total; x0 += gridDim.x * (256 * FLIGHT)) {
      uint32_t kw[FLIGHT], vw[FLIGHT], kf[FLIGHT], vf[FLIGHT];
#pragma unroll
      for (int y = 0; y < FLIGHT; ++y) {               // all loads first: their latency is what this kernel would wait for
        const unsigned x = x0 + y * 256, row_of = x / PIECES, i = row_of / d.heads;
        const int piece = x - row_of * PIECES, h = row_of - i * d.heads;
        const long long pos = first + i;
        kw[y] = vw[y] = kf[y] = vf[y] = 0;
        if (x < total && pos >= 0 && pos < d.capacity) {
          int slot = s;
          if (pages) slot = pages[(long long)s * (d.capacity / PAGE) + pos / PAGE];
          if (slot < 0 || slot >= d.slots) kf[y] = vf[y] = 0x7f;
          else {
            const long long row = (long long)h * d.capacity + pos;
            const long long c = cl + slot * d.code_slot + row * (HD / 2) + piece * (N / 2), f = fl + slot * d.scale_slot + row * NB + piece * N / BLOCK;
            if (N == 8) { kw[y] = *reinterpret_cast<const uint32_t*>(d.kc + c); vw[y] = *reinterpret_cast<const uint32_t*>(d.vc + c); }
            else { kw[y] = *reinterpret_cast<const uint16_t*>(d.kc + c); vw[y] = *reinterpret_cast<const uint16_t*>(d.vc + c); }
            kf[y] = d.ks[f]; vf[y] = d.vs[f];
          }
        }
      }
#pragma unroll
      for (int y = 0; y < FLIGHT; ++y) {
        const unsigned x = x0 + y * 256, row_of = x / PIECES, i = row_of / d.heads;
        const int piece = x - row_of * PIECES, h = row_of - i * d.heads;
        if (x >= total) break;
        const float ks = e4m3_f32(kf[y]) * pow2(d.k_exp), vs = e4m3_f32(vf[y]) * pow2(d.v_exp);
        float kx[N], vx[N];
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          const float2 a = f16x2_f32(e2m1x2_f16x2((kw[y] >> (8 * j)) & 0xff)), b = f16x2_f32(e2m1x2_f16x2((vw[y] >> (8 * j)) & 0xff));
          kx[2 * j] = a.x * ks; kx[2 * j + 1] = a.y * ks;
          vx[2 * j] = b.x * vs; vx[2 * j + 1] = b.y * vs;
        }
        T* const kp = ko + l * out_layer + s * sk.b + i * sk.t + h * sk.h + piece * N;
        T* const vp = vo + l * out_layer + s * sv.b + i * sv.t + h * sv.h + piece * N;
        if (VEC) {
          Pack<T> a, b;
#pragma unroll
          for (int j = 0; j < N; ++j) { a.v[j] = kx[j]; b.v[j] = vx[j]; }
          a.store(kp); b.store(vp);
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) { kp[j] = from_f<T>(kx[j]); vp[j] = from_f<T>(vx[j]); }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- reorder
__device__ __forceinline__ int parent_of(const int* parents, int item, int j, int K) {
  const int p = parents[(long long)item * K + j];
  return p < 0 || p >= K ? j : p;
}
__device__ __forceinline__ int length_of(const int* lens, int slot, int capacity) { return min(max(lens[slot], 0), capacity); }

struct Kv4Page { long long codes, scales; int tokens, source; };      // offsets in bytes, tokens in use, and for a copy the beam it is of
// The page that is being filled: its used part is contiguous in each of the four tensors.  A thread takes the same 16 bytes of every beam's page
// that is somebody's parent into a column of shared memory of its own, then gives every beam with another parent its parent's.  So no
// thread waits for another, and everything is read before it is written: other threads write other bytes.  Blocks share an item's heads and layers.
__global__ void __launch_bounds__(128, 12) kv4_reorder_kernel(const Kv4Desc d, const int* __restrict__ lens, const int* __restrict__ parents, int K) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ uint4 buf[];                       // a piece of each source for every thread
  __shared__ Kv4Page from[64], to[64];                 // the pages that are read, and those that are written
  __shared__ int place_of[64], n_from, n_to, longest;
  const int item = blockIdx.x;
  const int cb = d.head_size / 2, sb = d.head_size / BLOCK;
  if (threadIdx.x == 0) n_from = n_to = longest = 0;
  for (int j = threadIdx.x; j < K; j += blockDim.x) place_of[j] = -1;
  __syncthreads();
  auto page_of = [&](int j, int n) {                   // where beam j keeps the page in which n tokens end, from the item's first slot on
    const long long before = (long long)(n / PAGE) * PAGE;
    return Kv4Page{j * d.code_slot + before * cb, j * d.scale_slot + before * sb, n % PAGE, 0};
  };
  for (int j = threadIdx.x; j < K; j += blockDim.x) {
    const int p = parent_of(parents, item, j, K), n = length_of(lens, item * K + p, d.capacity);
    if (p == j || n % PAGE == 0) continue;
    if (atomicCAS(&place_of[p], -1, -2) == -1) {       // the first to name this parent
      const int i = atomicAdd(&n_from, 1);
      from[i] = page_of(p, n);
      atomicExch(&place_of[p], i);
    }
    Kv4Page w = page_of(j, n);
    w.source = p;
    to[atomicAdd(&n_to, 1)] = w;
    atomicMax(&longest, n % PAGE);
  }
  __syncthreads();
  const unsigned code_pieces = ceil_div(longest * cb, 16), scale_pieces = ceil_div(longest * sb, 16), half = code_pieces + scale_pieces;
  const unsigned all = d.layers * d.heads * 2 * half;
  for (unsigned x = blockIdx.y * blockDim.x + threadIdx.x; x < all; x += gridDim.y * blockDim.x) {
    const unsigned plane = x / (2 * half), layer = plane / d.heads, h = plane - layer * d.heads;
    unsigned y = x - plane * 2 * half;
    const bool is_v = y >= half;
    if (is_v) y -= half;
    const bool is_scale = y >= code_pieces;
    const int bytes = is_scale ? sb : cb, first = (is_scale ? y - code_pieces : y) * 16;           // bytes of a token; the piece's first byte
    uint8_t* const base = (is_scale ? (is_v ? d.vs : d.ks) + layer * d.scale_layer + item * K * d.scale_slot
                                    : (is_v ? d.vc : d.kc) + layer * d.code_layer + item * K * d.code_slot) + (long long)h * d.capacity * bytes + first;
    for (int j = 0; j < n_from; ++j)                   // asynchronous copies: all of them are in flight at once
      if (first < from[j].tokens * bytes)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&buf[j * blockDim.x + threadIdx.x])),
                     "l"(base + (is_scale ? from[j].scales : from[j].codes)) : "memory");
    asm volatile("cp.async.wait_all;" ::: "memory");   // a thread reads nothing but its own copies
    for (int j = 0; j < n_to; ++j) {
      const int keep = to[j].tokens * bytes - first;
      if (keep <= 0) continue;
      const uint4 val = buf[place_of[to[j].source] * blockDim.x + threadIdx.x];
      uint8_t* const a = base + (is_scale ? to[j].scales : to[j].codes);
      if (keep >= 16) *reinterpret_cast<uint4*>(a) = val;
      else {                                           // bytes behind the last token stay as they are
        const uint8_t* b = reinterpret_cast<const uint8_t*>(&val);
        for (int z = 0; z < keep; ++z) a[z] = b[z];
      }
    }
  }
}
// Page tables and lengths, behind the copies (which read the lengths): one block per item, a beam's column of entries at a time.
__global__ void __launch_bounds__(256) kv4_tables_kernel(int* __restrict__ pages, int* __restrict__ lens, const int* __restrict__ parents, int K, int n_pages, int capacity) {
  pdl_trigger();
  pdl_wait();
  __shared__ int new_len[64], src[64];
  __shared__ int buf[2048];
  const int item = blockIdx.x;
  if (threadIdx.x < K) {
    const int of = parent_of(parents, item, threadIdx.x, K);
    src[threadIdx.x] = of;
    new_len[threadIdx.x] = length_of(lens, item * K + of, capacity);
  }
  __syncthreads();
  if (threadIdx.x < K) lens[item * K + threadIdx.x] = new_len[threadIdx.x];
  const int per = 2048 / K;
  for (int p0 = 0; p0 < n_pages; p0 += per) {
    const int w = min(per, n_pages - p0);
    for (int t = threadIdx.x; t < w * K; t += 256) buf[t / w * per + t % w] = pages[(long long)(item * K + t / w) * n_pages + p0 + t % w];
    __syncthreads();
    for (int t = threadIdx.x; t < w * K; t += 256) {
      const int j = t / w, p = p0 + t % w;
      pages[(long long)(item * K + j) * n_pages + p] = p < new_len[j] / PAGE ? buf[src[j] * per + t % w] : item * K + j;
    }
    __syncthreads();
  }
}

inline bool aligned16(const void* p, const RowStrides& s, int elt) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(s.b * elt) | (uintptr_t)(s.t * elt) | (uintptr_t)(s.h * elt)) & 15) == 0;
}
inline unsigned at_most(long long blocks, long long most) { return (unsigned)(blocks < most ? blocks : most); }
#define KV4_HEADS(HD_VALUE, CALL)                                                                          \
  switch (HD_VALUE) {                                                                                      \
    case 32: { constexpr int HD = 32; return CALL; }                                                       \
    case 64: { constexpr int HD = 64; return CALL; }                                                       \
    case 80: { constexpr int HD = 80; return CALL; }                                                       \
    case 96: { constexpr int HD = 96; return CALL; }                                                       \
    case 128: { constexpr int HD = 128; return CALL; }                                                     \
    default: return LLMB_ERR_BAD_ARG;                                                                      \
  }

template <typename T, int HD>
int append(const Kv4Desc& d, int layer, const void* k, const void* v, const int* start, const int* counts, int n, RowStrides sk, RowStrides sv, cudaStream_t st) {
  constexpr int ROWS = 256 / AppendGroup<HD>::value;
  const long long rows = (long long)d.heads * n;
  if (rows > 0x7fffffffLL - (1 << 20)) return LLMB_ERR_BAD_ARG;
  const Divisor by_heads{(unsigned)d.heads, d.heads > 1 && (rows + (1 << 20)) * d.heads < 1LL << 32 ? (unsigned)(((1LL << 32) + d.heads - 1) / d.heads) : 0u};
  const dim3 grid(at_most(ceil_div_ll(rows, ROWS), ceil_div_ll((long long)sm_count() * 8, d.slots)), d.slots);
  const bool vec = aligned16(k, sk, sizeof(T)) && aligned16(v, sv, sizeof(T));
  return launch_pdl(vec ? kv4_append_kernel<T, HD, true> : kv4_append_kernel<T, HD, false>, grid, 256, 0, st, d, layer, (const T*)k, (const T*)v, start, counts, n, by_heads, sk, sv);
}
template <typename T, int HD>
int values(const Kv4Desc& d, int layer, void* k, void* v, const int* start, const int* pages, int n, long long out_layer, RowStrides sk, RowStrides sv, cudaStream_t st) {
  const long long total = (long long)n * d.heads * (HD * (int)sizeof(T) / 16), planes = (long long)(layer < 0 ? d.layers : 1) * d.slots;
  if (total > 0x7fffffffLL - (1 << 20) || planes > 0x7fffffffLL) return LLMB_ERR_BAD_ARG;
  const unsigned gy = at_most(planes, 65535);
  const dim3 grid(at_most(ceil_div_ll(total, 1024), ceil_div_ll((long long)sm_count() * 16, gy)), gy);
  const bool vec = aligned16(k, sk, sizeof(T)) && aligned16(v, sv, sizeof(T)) && (out_layer * (int)sizeof(T)) % 16 == 0;
  return launch_pdl(vec ? kv4_values_kernel<T, HD, true> : kv4_values_kernel<T, HD, false>, grid, 256, 0, st, d, layer, (T*)k, (T*)v, start, pages, n, out_layer, sk, sv);
}
}  // namespace

// The arguments of a call as the Python side (ops/kv4.py) packs them.
struct Kv4AppendArgs {
  const void *k, *v; const int *start, *counts;        // counts: optional
  long long kb, kt, kh, vb, vt, vh;
  int layer, n, dtype, pad;
};
struct Kv4ValuesArgs {
  void *k, *v; const int *start, *pages;               // pages: optional
  long long out_layer, kb, kt, kh, vb, vt, vh;         // layer -1: all layers, out_layer elements apart
  int layer, n, dtype, pad;
};

LLMB_API int llmb_kv4_append(const Kv4Desc* d, const Kv4AppendArgs* a, cudaStream_t st) {
  const RowStrides sk{a->kb, a->kt, a->kh}, sv{a->vb, a->vt, a->vh};
  if (a->dtype == LLMB_BF16) { KV4_HEADS(d->head_size, (append<__nv_bfloat16, HD>(*d, a->layer, a->k, a->v, a->start, a->counts, a->n, sk, sv, st))) }
  KV4_HEADS(d->head_size, (append<float, HD>(*d, a->layer, a->k, a->v, a->start, a->counts, a->n, sk, sv, st)))
}

LLMB_API int llmb_kv4_values(const Kv4Desc* d, const Kv4ValuesArgs* a, cudaStream_t st) {
  const RowStrides sk{a->kb, a->kt, a->kh}, sv{a->vb, a->vt, a->vh};
  if (a->dtype == LLMB_BF16) { KV4_HEADS(d->head_size, (values<__nv_bfloat16, HD>(*d, a->layer, a->k, a->v, a->start, a->pages, a->n, a->out_layer, sk, sv, st))) }
  KV4_HEADS(d->head_size, (values<float, HD>(*d, a->layer, a->k, a->v, a->start, a->pages, a->n, a->out_layer, sk, sv, st)))
}

struct Kv4ReorderArgs { int *pages, *lens; const int* parents; int K, pad; };

LLMB_API int llmb_kv4_reorder(const Kv4Desc* d, const Kv4ReorderArgs* a, cudaStream_t st) {
  int *pages = a->pages, *lens = a->lens, K = a->K;
  const int* parents = a->parents;
  const int items = K > 0 ? d->slots / K : 0;
  if (K < 1 || K > 64) return LLMB_ERR_BAD_ARG;
  const int threads = K <= 16 ? 128 : K <= 32 ? 64 : 32;        // at most 32 KB of pieces
  const long long pieces = (long long)d->layers * d->heads * 2 * (PAGE * (d->head_size / 2 + d->head_size / BLOCK) / 16);
  if (pieces > 0x7fffffffLL - (1 << 20)) return LLMB_ERR_BAD_ARG;
  const dim3 grid(items, at_most(ceil_div_ll(pieces, threads), ceil_div_ll((long long)sm_count() * 12, items)));
  int rc = launch_pdl(kv4_reorder_kernel, grid, threads, (size_t)K * threads * 16, st, *d, (const int*)lens, parents, K);
  if (rc) return rc;
  return launch_pdl(kv4_tables_kernel, items, 256, 0, st, pages, lens, parents, K, d->capacity / PAGE, d->capacity);
}
