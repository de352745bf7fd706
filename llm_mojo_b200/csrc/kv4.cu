// The 4-bit key/value cache (layout: kv4.cuh): rounding new keys and values into it, reading it back, and following a beam search.
//
// This file has no counterpart in the reference project, whose inference runs the whole forward pass for every token
// (infer_gpt2.mojo:56-144).
#include "kv4.cuh"
using namespace llmb;
using namespace kv4;

namespace {
struct RowStrides { long long b, t, h; };            // elements: sequence, token, head; the values of a head lie densely

// Sixteen values from p on, as floats; VEC: 16-byte loads.
template <typename T, bool VEC> __device__ __forceinline__ void load16(float (&x)[16], const T* p) {
  if (VEC) {
    constexpr int N = Pack<T>::N;
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) {
      Pack<T> v; v.load(p + i * N);
#pragma unroll
      for (int k = 0; k < N; ++k) x[i * N + k] = v.v[k];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = to_f<T>(p[k]);
  }
}
template <typename T, bool VEC> __device__ __forceinline__ void store16(T* p, const float (&x)[16]) {
  if (VEC) {
    constexpr int N = Pack<T>::N;
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) {
      Pack<T> v;
#pragma unroll
      for (int k = 0; k < N; ++k) v.v[k] = x[i * N + k];
      v.store(p + i * N);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) p[k] = from_f<T>(x[k]);
  }
}

// x / s correctly rounded from r = 1 / s correctly rounded: one step on the remainder (Markstein).  |x / s| stays far from both ends of fp32.
__device__ __forceinline__ float divide(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, s, x), r, q);
}

// One thread per block of 16 values; the threads of a row's key blocks and of its value blocks are neighbours (GROUP of them, some idle where
// 2 HD / 16 is no power of two) because a non-finite value in one block marks all of them.  Rows are counted (slot, head, token), the token
// fastest, so that a warp's stores are dense in the cache.
// The codes are those of the exact quotients x / s, s the scale.  A tie between two levels is a product of a midpoint's 3 bits and the scale's 4.
// The correctly rounded quotient is a midpoint only where x / s is one; a product with the rounded reciprocal is not (fl(1 / 0.875) 0.75 x 0.875
// lies above 0.75), and a true division costs eight operations against three.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4Desc d, int layer, const T* __restrict__ k, const T* __restrict__ v,
                                                         const int* __restrict__ start, const int* __restrict__ counts, int n, RowStrides sk, RowStrides sv) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = HD / BLOCK, GROUP = NB <= 2 ? 4 : NB <= 4 ? 8 : 16, ROWS = 256 / GROUP;
  const unsigned rows = (unsigned)d.slots * d.heads * n;        // below 2^31 (host)
  const int at = threadIdx.x % GROUP;
  const bool is_v = at >= NB;
  const int blk = is_v ? at - NB : at;
  const RowStrides st = is_v ? sv : sk;
  const T* const from = (is_v ? v : k) + blk * BLOCK;
  const int e = is_v ? d.v_exp : d.k_exp;
  const float unit = pow2(e), per_unit = pow2(-e);
  uint8_t* const codes = (is_v ? d.vc : d.kc) + layer * d.code_layer + blk * 8;
  uint8_t* const scales = (is_v ? d.vs : d.ks) + layer * d.scale_layer + blk;
  // whole groups walk the rows together, so the shuffles below have all their lanes
  for (unsigned r0 = blockIdx.x * ROWS; r0 < rows; r0 += gridDim.x * ROWS) {
    const unsigned r = r0 + threadIdx.x / GROUP, sh = r / (unsigned)n, s = sh / (unsigned)d.heads;
    const int i = (int)(r - sh * n), h = (int)(sh - s * d.heads);
    bool live = r < rows && at < 2 * NB;
    long long pos = 0;
    if (live) {
      pos = (long long)start[s] + i;
      live = pos >= 0 && pos < d.capacity && (counts == nullptr || i < counts[s]);
    }
    float x[16];
    float amax = 0.f;
    bool bad = false;
    if (live) {
      load16<T, VEC>(x, from + s * st.b + i * st.t + h * st.h);
#pragma unroll
      for (int j = 0; j < 16; ++j) { bad |= !(fabsf(x[j]) <= 3.402823466e38f); amax = fmaxf(amax, fabsf(x[j])); }
    }
#pragma unroll
    for (int o = 1; o < GROUP; o <<= 1) bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
    if (!live) continue;
    const uint32_t sc = e4m3(__fdiv_rn(amax * per_unit, 6.0f));
    const float s32 = e4m3_f32(sc) * unit, inv = __frcp_rn(s32);
    uint32_t lo = 0, hi = 0;
    if (!bad && sc != 0) {
      if (sc == 0x7e) {                                // the largest scale: what saturates stays in range
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = fminf(fmaxf(x[j], -8.f * s32), 8.f * s32);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = divide(x[j], s32, inv);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo |= e2m1x2(x[2 * j], x[2 * j + 1]) << (8 * j);
        hi |= e2m1x2(x[8 + 2 * j], x[9 + 2 * j]) << (8 * j);
      }
    }
    const long long row = (long long)h * d.capacity + pos;
    *reinterpret_cast<uint2*>(codes + s * d.code_slot + row * (HD / 2)) = make_uint2(lo, hi);
    scales[s * d.scale_slot + row * NB] = bad ? 0x7f : (uint8_t)sc;
  }
}

// One thread per 16 bytes of an output, of both the key and the value; the pieces of a row, then its heads, then its tokens are neighbours: the
// stores, which are most of the bytes, are dense where the outputs are.  A block stays with one slot of one layer.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(256) kv4_values_kernel(const Kv4Desc d, int layer, T* __restrict__ ko, T* __restrict__ vo, const int* __restrict__ start,
                                                         const int* __restrict__ pages, int n, long long out_layer, RowStrides sk, RowStrides sv) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = HD / BLOCK, N = 16 / sizeof(T), PIECES = HD / N;
  const unsigned total = (unsigned)n * d.heads * PIECES, planes = (layer < 0 ? d.layers : 1) * d.slots;      // below 2^31 (host)
  for (unsigned plane = blockIdx.y; plane < planes; plane += gridDim.y) {
    const int l = plane / d.slots, s = plane - l * d.slots;
    const long long first = start[s];
    const long long cl = (layer < 0 ? l : layer) * d.code_layer, fl = (layer < 0 ? l : layer) * d.scale_layer;
    for (unsigned x = blockIdx.x * 256 + threadIdx.x; x < total; x += gridDim.x * 256) {
      const unsigned row_of = x / PIECES, i = row_of / d.heads;
      const int piece = x - row_of * PIECES, h = row_of - i * d.heads;
      const long long pos = first + i;
      float kx[N], vx[N];
      float ks = 0.f, vs = 0.f;
      uint32_t kw = 0, vw = 0;
      if (pos >= 0 && pos < d.capacity) {
        int slot = s;
        if (pages) slot = pages[(long long)s * (d.capacity / PAGE) + pos / PAGE];
        if (slot < 0 || slot >= d.slots) ks = vs = __int_as_float(0x7fc00000);
        else {
          const long long row = (long long)h * d.capacity + pos;
          const long long c = cl + slot * d.code_slot + row * (HD / 2) + piece * (N / 2), f = fl + slot * d.scale_slot + row * NB + piece * N / BLOCK;
          if (N == 8) { kw = *reinterpret_cast<const uint32_t*>(d.kc + c); vw = *reinterpret_cast<const uint32_t*>(d.vc + c); }
          else { kw = *reinterpret_cast<const uint16_t*>(d.kc + c); vw = *reinterpret_cast<const uint16_t*>(d.vc + c); }
          ks = e4m3_f32(d.ks[f]) * pow2(d.k_exp); vs = e4m3_f32(d.vs[f]) * pow2(d.v_exp);
        }
      }
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        const float2 a = f16x2_f32(e2m1x2_f16x2((kw >> (8 * j)) & 0xff)), b = f16x2_f32(e2m1x2_f16x2((vw >> (8 * j)) & 0xff));
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

// ---------------------------------------------------------------------------------------------- reorder
__device__ __forceinline__ int parent_of(const int* parents, int item, int j, int K) {
  const int p = parents[(long long)item * K + j];
  return p < 0 || p >= K ? j : p;
}
__device__ __forceinline__ int length_of(const int* lens, int slot, int capacity) { return min(max(lens[slot], 0), capacity); }

// The page that is being filled: its used part is contiguous in each of the four tensors.  One block per (item, head, layer); a thread takes the
// same 16 bytes of every beam's page that is somebody's parent into a column of shared memory of its own, then gives every beam with another
// parent its parent's.  So no thread waits for another, and everything is read before it is written: other threads write other bytes.
constexpr int REORDER_PIECES = 2048;                  // 16-byte pieces in shared memory: one of each beam for every thread
__global__ void __launch_bounds__(256) kv4_reorder_kernel(const Kv4Desc d, const int* __restrict__ lens, const int* __restrict__ parents, int K) {
  pdl_trigger();
  pdl_wait();
  __shared__ uint4 buf[REORDER_PIECES];
  __shared__ int of[64], len[64], wanted[64];
  const int item = blockIdx.x, h = blockIdx.y, layer = blockIdx.z, j0 = threadIdx.x;
  for (int j = j0; j < K; j += blockDim.x) { of[j] = parent_of(parents, item, j, K); len[j] = length_of(lens, item * K + j, d.capacity); wanted[j] = 0; }
  __syncthreads();
  for (int j = j0; j < K; j += blockDim.x) if (of[j] != j && len[of[j]] % PAGE) wanted[of[j]] = 1;
  __syncthreads();
  const int cb = d.head_size / 2, sb = d.head_size / BLOCK, code_pieces = PAGE * cb / 16, scale_pieces = PAGE * sb / 16;
  for (int x = threadIdx.x; x < 2 * (code_pieces + scale_pieces); x += blockDim.x) {
    const int y = x < code_pieces + scale_pieces ? x : x - code_pieces - scale_pieces;
    const bool is_v = y != x, is_scale = y >= code_pieces;
    const int bytes = is_scale ? sb : cb, first = (is_scale ? y - code_pieces : y) * 16;           // bytes of a token; the piece's first byte
    const long long slot_stride = is_scale ? d.scale_slot : d.code_slot;
    uint8_t* const base = (is_scale ? (is_v ? d.vs : d.ks) + layer * d.scale_layer : (is_v ? d.vc : d.kc) + layer * d.code_layer) +
                          item * K * slot_stride + (long long)h * d.capacity * bytes + first;
    auto place = [&](int j, int n) { return base + j * slot_stride + (long long)(n / PAGE) * PAGE * bytes; };
    for (int j = 0; j < K; ++j)
      if (wanted[j] && first < (len[j] % PAGE) * bytes) buf[j * blockDim.x + threadIdx.x] = *reinterpret_cast<const uint4*>(place(j, len[j]));
    for (int j = 0; j < K; ++j) {
      const int p = of[j], n = len[p], keep = (n % PAGE) * bytes - first;
      if (p == j || keep <= 0) continue;
      const uint4 val = buf[p * blockDim.x + threadIdx.x];
      uint8_t* const a = place(j, n);
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
  constexpr int NB = HD / BLOCK, GROUP = NB <= 2 ? 4 : NB <= 4 ? 8 : 16;
  const long long rows = (long long)d.slots * d.heads * n;
  if (rows > 0x7fffffffLL - (1 << 20)) return LLMB_ERR_BAD_ARG;
  const unsigned grid = at_most(ceil_div_ll(rows * GROUP, 256), (long long)sm_count() * 8);
  const bool vec = aligned16(k, sk, sizeof(T)) && aligned16(v, sv, sizeof(T));
  return launch_pdl(vec ? kv4_append_kernel<T, HD, true> : kv4_append_kernel<T, HD, false>, grid, 256, 0, st, d, layer, (const T*)k, (const T*)v, start, counts, n, sk, sv);
}
template <typename T, int HD>
int values(const Kv4Desc& d, int layer, void* k, void* v, const int* start, const int* pages, int n, long long out_layer, RowStrides sk, RowStrides sv, cudaStream_t st) {
  const long long total = (long long)n * d.heads * (HD * (int)sizeof(T) / 16), planes = (long long)(layer < 0 ? d.layers : 1) * d.slots;
  if (total > 0x7fffffffLL - (1 << 20) || planes > 0x7fffffffLL) return LLMB_ERR_BAD_ARG;
  const unsigned gy = at_most(planes, 65535);
  const dim3 grid(at_most(ceil_div_ll(total, 256), ceil_div_ll((long long)sm_count() * 16, gy)), gy);
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

LLMB_API int llmb_kv4_reorder(const Kv4Desc* d, int* pages, int* lens, const int* parents, int K, cudaStream_t st) {
  const int items = K > 0 ? d->slots / K : 0;
  if (K < 1 || K > 64 || d->layers > 65535 || d->heads > 65535) return LLMB_ERR_BAD_ARG;
  int rc = launch_pdl(kv4_reorder_kernel, dim3(items, d->heads, d->layers), K <= 8 ? 256 : REORDER_PIECES / K / 32 * 32, 0, st, *d, (const int*)lens, parents, K);
  if (rc) return rc;
  return launch_pdl(kv4_tables_kernel, items, 256, 0, st, pages, lens, parents, K, d->capacity / PAGE, d->capacity);
}
