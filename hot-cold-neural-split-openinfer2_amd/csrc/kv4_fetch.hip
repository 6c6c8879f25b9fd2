// Positions of the 4-bit KV cache's rows as dense k and v: what its codes stand
// for.
//
// One launch.  Every workgroup makes the rows' prefix sums for itself, in LDS (a
// launch of its own for them would cost more than they do), and then takes
// every so-many-th set of 16 tokens; a wave has four tokens, 16 lanes and 8 dims a
// lane each, and goes over kv heads, which is how the append writes them.
#include "capi_util.h"
#include "kv4.h"
#include "rotary.h"

namespace oi2 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct FetchArgs {
  const int32_t *table, *lens, *first, *count;
  int32_t* cu;
  int n_seqs, width, max_len, n_pages, n_kv, max_tokens;
  int heads_each, chunks;     // kv heads of a wave's turn, and how many turns a token's heads take
  int zero, wide;             // wide: 16-byte stores
  const uint8_t* pages;       // of the layer
  void* dst[2];               // k, v
  int64_t token_stride[2], head_stride[2];
};

// 8 values over s, in fp16 pairs (exact).
__device__ __forceinline__ void values8(f16x2 (&y)[4], uint32_t d, uint16_t scale) {
  const _Float16 s = __builtin_bit_cast(_Float16, scale);
  const f16x2 ss = {s, s};
  const uint32_t lo = low4(d), hi = high4(d);
  y[0] = whole2(lo, false) * ss;
  y[1] = whole2(lo, true) * ss;
  y[2] = whole2(hi, false) * ss;
  y[3] = whole2(hi, true) * ss;
}

// DTYPE: OI2_DTYPE_*.
template <int DTYPE>
__device__ __forceinline__ void store8(void* base, int64_t at, const f16x2 (&y)[4], bool wide) {
  if constexpr (DTYPE == OI2_DTYPE_F32) {
    float* p = static_cast<float*>(base) + at;
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = (float)y[e / 2][e % 2];
    if (wide) {
      *reinterpret_cast<f32x4*>(p) = f32x4{z[0], z[1], z[2], z[3]};
      *reinterpret_cast<f32x4*>(p + 4) = f32x4{z[4], z[5], z[6], z[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = z[e];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    uint32_t z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      z[e] = DTYPE == OI2_DTYPE_F16 ? __builtin_bit_cast(uint32_t, y[e])
                                    : narrow<true>((float)y[e][0]) | (uint32_t)narrow<true>((float)y[e][1]) << 16;
    if (wide) {
      *reinterpret_cast<u32x4*>(p) = u32x4{z[0], z[1], z[2], z[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[2 * e] = (uint16_t)z[e];
        p[2 * e + 1] = (uint16_t)(z[e] >> 16);
      }
    }
  }
}

constexpr uint32_t kMost = 0x7FFFFFFF;
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kMost); }

template <int DTYPE>
__global__ __launch_bounds__(kThreads) void k_kv4_fetch(FetchArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ uint32_t s_wave[kWaves];
  const int n = a.n_seqs, tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
  int32_t* s_end = lds;              // inclusive sums of the rows' tokens
  int32_t* s_first = s_end + n;      // first position that is read
  const int per = (n + kThreads - 1) / kThreads, r0 = min(tid * per, n), r1 = min(r0 + per, n);
  uint32_t mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int len = min(max(a.lens[r], 0), a.max_len), f = a.first ? min(max(a.first[r], 0), len) : 0;
    const int count = min(max(a.count[r], 0), len - f);
    s_first[r] = f;
    mine = add_sat(mine, (uint32_t)count);
    s_end[r] = (int)mine;
  }
  uint32_t before = mine;            // of the wave's lanes up to this one
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t x = (uint32_t)__shfl_up((int)before, d);
    if (lane >= d) before = add_sat(before, x);
  }
  if (lane == 63) s_wave[wave] = before;
  uint32_t base = (uint32_t)__shfl_up((int)before, 1);
  if (lane == 0) base = 0;
  __syncthreads();
  for (int w = 0; w < wave; ++w) base = add_sat(base, s_wave[w]);
  for (int r = r0; r < r1; ++r) s_end[r] = (int)add_sat((uint32_t)s_end[r], base);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int r = tid; r <= n; r += kThreads) a.cu[r] = r ? s_end[r - 1] : 0;
  const int total = min(s_end[n - 1], a.max_tokens), tokens = a.zero ? a.max_tokens : total;

  const int u = lane & 15;
  const int64_t tasks = ((int64_t)tokens + 3) / 4 * a.chunks;
  for (int64_t task = (int64_t)blockIdx.x * kWaves + wave; task < tasks; task += (int64_t)gridDim.x * kWaves) {
    const int64_t quad = task / a.chunks;
    const int g0 = (int)(task - quad * a.chunks) * a.heads_each, g1 = min(g0 + a.heads_each, a.n_kv);
    const int64_t t = 4 * quad + (lane >> 4);
    if (t >= tokens) continue;
    int64_t at[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) at[w] = t * a.token_stride[w] + 8 * u;
    if (t >= total) {
      const f16x2 none[4] = {};
      for (int g = g0; g < g1; ++g)
#pragma unroll
        for (int w = 0; w < 2; ++w) store8<DTYPE>(a.dst[w], at[w] + g * a.head_stride[w], none, a.wide);
      continue;
    }
    int lo = 0, hi = n - 1;          // the first row that ends past t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_end[mid] > t) hi = mid;
      else lo = mid + 1;
    }
    const int pos = s_first[lo] + (int)t - (lo ? s_end[lo - 1] : 0), p = pos % kPage;
    int id = a.table[(int64_t)lo * a.width + pos / kPage];
    id = (unsigned)id < (unsigned)a.n_pages ? id : 0;       // a damaged table reads page 0
    const uint8_t* block = a.pages + (int64_t)id * a.n_kv * k4Block;
#pragma unroll 4
    for (int g = g0; g < g1; ++g) {
      const uint8_t* b = block + (int64_t)g * k4Block;
      const uint32_t kd = *reinterpret_cast<const uint32_t*>(b + k4_at(p, u)), vd = *reinterpret_cast<const uint32_t*>(b + v4_at(p, u));
      const uint16_t ks = *reinterpret_cast<const uint16_t*>(b + k4_scale_at(p, u / 4));
      const uint16_t vs = *reinterpret_cast<const uint16_t*>(b + v4_scale_at(p, u / 4));
      f16x2 y[4];
      values8(y, kd, ks);
      store8<DTYPE>(a.dst[0], at[0] + g * a.head_stride[0], y, a.wide);
      values8(y, vd, vs);
      store8<DTYPE>(a.dst[1], at[1] + g * a.head_stride[1], y, a.wide);
    }
  }
}

// Whether no two of the (tokens, heads, 128) values at h share memory.
bool apart(const oi2_heads* h, int64_t tokens) {
  const int64_t st = h->token_stride, sh = h->head_stride, nh = h->heads;
  if (st < 0 || sh < 0) return false;
  if (tokens <= 1) return nh <= 1 || sh >= kHeadD;
  if (nh <= 1) return st >= kHeadD;
  return (sh >= kHeadD && st >= (nh - 1) * sh + kHeadD) || (st >= kHeadD && sh >= (tokens - 1) * st + kHeadD);
}

// Whether those at k and at v do: where their spans meet, only values that lie
// alike, one behind the other within a token, are taken for apart.
bool meet(const oi2_heads* k, const oi2_heads* v, int64_t tokens, int size) {
  auto span = [&](const oi2_heads* h) { return ((tokens - 1) * h->token_stride + (h->heads - 1) * h->head_stride + kHeadD) * size; };
  const uintptr_t a = (uintptr_t)k->data, b = (uintptr_t)v->data;
  if (a + span(k) <= b || b + span(v) <= a) return false;
  if (k->token_stride != v->token_stride || k->head_stride != v->head_stride || a == b) return true;
  const int64_t apart = (int64_t)(a < b ? b - a : a - b), one = ((k->heads - 1) * k->head_stride + kHeadD) * size;
  return apart < one || (tokens > 1 && apart + one > k->token_stride * size);
}

}  // namespace
}  // namespace oi2

using namespace oi2;

extern "C" int oi2_kv4_fetch(const oi2_paged* c, int32_t layer, const int32_t* first, const int32_t* count, int32_t dtype,
                             int32_t max_tokens, const oi2_heads* k, const oi2_heads* v, int32_t* cu, void* stream) {
  clear_error();
  if (int rc = check_paged4(c, layer)) return rc;
  const bool zero = dtype & OI2_ZERO_LEFT_OUT;
  dtype &= ~OI2_ZERO_LEFT_OUT;
  OI2_CHECK_ARG(dtype == OI2_DTYPE_F16 || dtype == OI2_DTYPE_BF16 || dtype == OI2_DTYPE_F32, "dtype %d: fp16, bf16 or fp32", dtype);
  OI2_CHECK_ARG(max_tokens >= 0, "%d tokens", max_tokens);
  OI2_CHECK_ARG(count && cu, "null counts or sums");
  OI2_CHECK_ARG(k && v && k->heads == c->n_kv && v->heads == c->n_kv, "k and v need the cache's %d heads", c->n_kv);
  FetchArgs a{};
  if (max_tokens) {
    const int size = dtype == OI2_DTYPE_F32 ? 4 : 2;
    const oi2_heads* out[2] = {k, v};
    a.wide = 1;
    for (int w = 0; w < 2; ++w) {
      OI2_CHECK_ARG(out[w]->data && (uintptr_t)out[w]->data % size == 0, "k and v must be non-null and aligned");
      OI2_CHECK_ARG(apart(out[w], max_tokens), "values of an output share memory");
      a.dst[w] = const_cast<void*>(out[w]->data);
      a.token_stride[w] = out[w]->token_stride;
      a.head_stride[w] = out[w]->head_stride;
      if ((uintptr_t)out[w]->data % 16 || out[w]->token_stride * size % 16 || out[w]->head_stride * size % 16) a.wide = 0;
    }
    OI2_CHECK_ARG(!meet(k, v, max_tokens, size), "k and v share memory");
  }
  a.table = c->block_table;
  a.lens = c->lens;
  a.first = first;
  a.count = count;
  a.cu = cu;
  a.n_seqs = c->n_seqs;
  a.max_len = c->max_len;
  a.width = (c->max_len + kPage - 1) / kPage;
  a.n_pages = c->n_pages;
  a.n_kv = c->n_kv;
  a.max_tokens = max_tokens;
  a.zero = zero;
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * k4Block;
  a.heads_each = c->n_kv < 4 ? c->n_kv : 4;
  a.chunks = (c->n_kv + a.heads_each - 1) / a.heads_each;
  const int64_t want = (((int64_t)max_tokens + 3) / 4 * a.chunks + kWaves - 1) / kWaves;
  const uint32_t groups = (uint32_t)(want < 1 ? 1 : want < 2048 ? want : 2048);
  const size_t lds = (size_t)c->n_seqs * 8;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(groups), block(kThreads);
  if (dtype == OI2_DTYPE_F16) hipLaunchKernelGGL(k_kv4_fetch<OI2_DTYPE_F16>, grid, block, lds, st, a);
  else if (dtype == OI2_DTYPE_BF16) hipLaunchKernelGGL(k_kv4_fetch<OI2_DTYPE_BF16>, grid, block, lds, st, a);
  else hipLaunchKernelGGL(k_kv4_fetch<OI2_DTYPE_F32>, grid, block, lds, st, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}
