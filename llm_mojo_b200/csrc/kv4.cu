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

// One thread per block of 16 values; the threads of a row's key blocks and of its value blocks are neighbours (GROUP of them, some idle where
// 2 HD / 16 is no power of two) because a non-finite value in one block marks all of them.  Rows are counted (slot, head, token), the token
// fastest, so that a warp's stores are dense in the cache.  The quotients are true divisions: x / scale is then a tie between two levels exactly
// where it is one in the reals (a midpoint has 3 bits, a scale 4, so x would have to be their product), and the conversion rounds it to even.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4Desc d, int layer, const T* __restrict__ k, const T* __restrict__ v,
                                                         const int* __restrict__ start, const int* __restrict__ counts, int n, RowStrides sk, RowStrides sv) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = HD / BLOCK, GROUP = NB <= 2 ? 4 : NB <= 4 ? 8 : 16;
  const long long rows = (long long)d.slots * d.heads * n;
  const int at = threadIdx.x % GROUP;
  const bool is_v = at >= NB;
  const int blk = is_v ? at - NB : at;
  // whole groups walk the rows together, so the shuffles below have all their lanes
  for (long long r0 = (long long)blockIdx.x * (256 / GROUP); r0 < rows; r0 += (long long)gridDim.x * (256 / GROUP)) {
    const long long r = r0 + threadIdx.x / GROUP;
    const int i = (int)(r % n);
    const long long sh = r / n;
    const int h = (int)(sh % d.heads), s = (int)(sh / d.heads);
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
      const RowStrides& st = is_v ? sv : sk;
      load16<T, VEC>(x, (is_v ? v : k) + s * st.b + i * st.t + h * st.h + blk * BLOCK);
#pragma unroll
      for (int j = 0; j < 16; ++j) { bad |= !(fabsf(x[j]) <= 3.402823466e38f); amax = fmaxf(amax, fabsf(x[j])); }
    }
#pragma unroll
    for (int o = 1; o < GROUP; o <<= 1) bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
    if (!live) continue;
    const int e = is_v ? d.v_exp : d.k_exp;
    const uint32_t sc = e4m3(__fdiv_rn(amax * pow2(-e), 6.0f));
    const float s32 = e4m3_f32(sc) * pow2(e);
    uint32_t lo = 0, hi = 0;
    if (!bad && sc != 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo |= e2m1x2(__fdiv_rn(x[2 * j], s32), __fdiv_rn(x[2 * j + 1], s32)) << (8 * j);
        hi |= e2m1x2(__fdiv_rn(x[8 + 2 * j], s32), __fdiv_rn(x[9 + 2 * j], s32)) << (8 * j);
      }
    }
    const long long row = (long long)h * d.capacity + pos;
    uint8_t* codes = (is_v ? d.vc : d.kc) + layer * d.code_layer + s * d.code_slot + row * (HD / 2) + blk * 8;
    uint8_t* scales = (is_v ? d.vs : d.ks) + layer * d.scale_layer + s * d.scale_slot + row * NB + blk;
    *reinterpret_cast<uint2*>(codes) = make_uint2(lo, hi);
    *scales = bad ? 0x7f : (uint8_t)sc;
  }
}

// One thread per block of 16 values of both the key and the value; the blocks of a row, then its heads, then its tokens are neighbours, so
// that the stores, which are most of the bytes, are dense where the outputs are.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(256) kv4_values_kernel(const Kv4Desc d, int layer, T* __restrict__ ko, T* __restrict__ vo, const int* __restrict__ start,
                                                         const int* __restrict__ pages, int n, long long out_layer, RowStrides sk, RowStrides sv) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = HD / BLOCK;
  const int layers = layer < 0 ? d.layers : 1;
  const long long total = (long long)layers * d.slots * n * d.heads * NB;
  for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < total; x += (long long)gridDim.x * 256) {
    const int blk = (int)(x % NB);
    long long r = x / NB;
    const int h = (int)(r % d.heads); r /= d.heads;
    const int i = (int)(r % n); r /= n;
    const int s = (int)(r % d.slots), l = (int)(r / d.slots);
    const long long pos = (long long)start[s] + i;
    float kx[16], vx[16];
    if (pos < 0 || pos >= d.capacity) {
#pragma unroll
      for (int j = 0; j < 16; ++j) kx[j] = vx[j] = 0.f;
    } else {
      int slot = s;
      if (pages) slot = pages[(long long)s * (d.capacity / PAGE) + pos / PAGE];
      if (slot < 0 || slot >= d.slots) {
#pragma unroll
        for (int j = 0; j < 16; ++j) kx[j] = vx[j] = __int_as_float(0x7fc00000);
      } else {
        const long long row = (long long)h * d.capacity + pos;
        const long long c = (layer < 0 ? l : layer) * d.code_layer + slot * d.code_slot + row * (HD / 2) + blk * 8;
        const long long f = (layer < 0 ? l : layer) * d.scale_layer + slot * d.scale_slot + row * NB + blk;
        const uint2 kc = *reinterpret_cast<const uint2*>(d.kc + c), vc = *reinterpret_cast<const uint2*>(d.vc + c);
        const float ks = e4m3_f32(d.ks[f]) * pow2(d.k_exp), vs = e4m3_f32(d.vs[f]) * pow2(d.v_exp);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 a = f16x2_f32(e2m1x2_f16x2(((j < 4 ? kc.x : kc.y) >> (8 * (j & 3))) & 0xff));
          const float2 b = f16x2_f32(e2m1x2_f16x2(((j < 4 ? vc.x : vc.y) >> (8 * (j & 3))) & 0xff));
          kx[2 * j] = a.x * ks; kx[2 * j + 1] = a.y * ks;
          vx[2 * j] = b.x * vs; vx[2 * j + 1] = b.y * vs;
        }
      }
    }
    store16<T, VEC>(ko + l * out_layer + s * sk.b + i * sk.t + h * sk.h + blk * BLOCK, kx);
    store16<T, VEC>(vo + l * out_layer + s * sv.b + i * sv.t + h * sv.h + blk * BLOCK, vx);
  }
}

// ---------------------------------------------------------------------------------------------- reorder
__device__ __forceinline__ int parent_of(const int* parents, int item, int j, int K) {
  const int p = parents[(long long)item * K + j];
  return p < 0 || p >= K ? j : p;
}
__device__ __forceinline__ int length_of(const int* lens, int slot, int capacity) { return min(max(lens[slot], 0), capacity); }

// The page that is being filled: one block per (item, head, layer) takes 16-byte pieces of every beam's page into shared memory, then every beam
// that has another parent writes its parent's.  Beams of an item are read before any of them is written; items, heads and layers do not meet.
constexpr int REORDER_THREADS = 256;
__global__ void __launch_bounds__(REORDER_THREADS) kv4_reorder_kernel(const Kv4Desc d, const int* __restrict__ lens, const int* __restrict__ parents, int K) {
  pdl_trigger();
  pdl_wait();
  constexpr int PIECES = 512;                          // 16-byte pieces in shared memory at a time
  __shared__ uint4 buf[PIECES];
  const int item = blockIdx.x, h = blockIdx.y, layer = blockIdx.z;
  const int cb = d.head_size / 2, sb = d.head_size / BLOCK;
  // pieces of one beam's page: codes and scales of keys, then of values (all multiples of 16 bytes for 64 tokens)
  const int code_pieces = PAGE * cb / 16, scale_pieces = PAGE * sb / 16, all = 2 * (code_pieces + scale_pieces);
  const int per = PIECES / K;                          // pieces of each beam at a time (K <= 64)
  auto address = [&](int slot, int page, int x, int* token) -> uint8_t* {
    const bool is_v = x >= code_pieces + scale_pieces;
    if (is_v) x -= code_pieces + scale_pieces;
    const bool is_scale = x >= code_pieces;
    if (is_scale) x -= code_pieces;
    const int bytes = is_scale ? sb : cb;
    *token = x * 16 / bytes;                           // the first token that has a byte in the piece
    uint8_t* base = is_scale ? (is_v ? d.vs : d.ks) + layer * d.scale_layer + slot * d.scale_slot : (is_v ? d.vc : d.kc) + layer * d.code_layer + slot * d.code_slot;
    return base + ((long long)h * d.capacity + (long long)page * PAGE) * bytes + x * 16;
  };
  for (int x0 = 0; x0 < all; x0 += per) {
    const int w = min(per, all - x0);
    for (int t = threadIdx.x; t < w * K; t += REORDER_THREADS) {
      const int j = t / w, x = x0 + t % w, slot = item * K + j;
      const int len = length_of(lens, slot, d.capacity);
      int token;
      if (len % PAGE == 0) continue;
      uint8_t* a = address(slot, len / PAGE, x, &token);
      if (token < len % PAGE) buf[j * per + t % w] = *reinterpret_cast<const uint4*>(a);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < w * K; t += REORDER_THREADS) {
      const int j = t / w, x = x0 + t % w, of = parent_of(parents, item, j, K);
      const int len = length_of(lens, item * K + of, d.capacity), rest = len % PAGE;
      if (of == j || rest == 0) continue;
      int token;
      uint8_t* a = address(item * K + j, len / PAGE, x, &token);
      if (token >= rest) continue;
      // a piece of scales may hold tokens behind the last one: those stay as they are
      const bool is_scale = x % (code_pieces + scale_pieces) >= code_pieces;
      const int bytes = is_scale ? sb : cb;
      const int first = (x % (code_pieces + scale_pieces) - (is_scale ? code_pieces : 0)) * 16, keep = rest * bytes - first;
      const uint4 val = buf[of * per + t % w];
      if (keep >= 16) *reinterpret_cast<uint4*>(a) = val;
      else {
        const uint8_t* b = reinterpret_cast<const uint8_t*>(&val);
        for (int y = 0; y < keep; ++y) a[y] = b[y];
      }
    }
    __syncthreads();
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
inline unsigned grid_of(long long threads) {
  const long long blocks = ceil_div_ll(threads, 256), most = (long long)sm_count() * 16;
  return (unsigned)(blocks < most ? blocks : most);
}
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
  const unsigned grid = grid_of((long long)d.slots * d.heads * n * GROUP);
  const bool vec = aligned16(k, sk, sizeof(T)) && aligned16(v, sv, sizeof(T));
  return launch_pdl(vec ? kv4_append_kernel<T, HD, true> : kv4_append_kernel<T, HD, false>, grid, 256, 0, st, d, layer, (const T*)k, (const T*)v, start, counts, n, sk, sv);
}
template <typename T, int HD>
int values(const Kv4Desc& d, int layer, void* k, void* v, const int* start, const int* pages, int n, long long out_layer, RowStrides sk, RowStrides sv, cudaStream_t st) {
  const unsigned grid = grid_of((long long)(layer < 0 ? d.layers : 1) * d.slots * n * d.heads * (HD / BLOCK));
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
  int rc = launch_pdl(kv4_reorder_kernel, dim3(items, d->heads, d->layers), REORDER_THREADS, 0, st, *d, (const int*)lens, parents, K);
  if (rc) return rc;
  return launch_pdl(kv4_tables_kernel, items, 256, 0, st, pages, lens, parents, K, d->capacity / PAGE, d->capacity);
}
