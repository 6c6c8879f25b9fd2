// Positions of the 4-bit KV cache's rows as dense k and v: what its codes stand
// for.
//
// One launch.  Every workgroup makes the rows' prefix sums for itself, in LDS (a
// launch of its own for them would cost more than they do), and then takes
// pages of one kv head, every so-many-th of what is read: what lies in a line of
// memory, or in a page's scales, is read by one workgroup.  A turn is a chain of a
// search of the sums in LDS, the table's entry, the page and the stores.
//
// Bound by its bytes: 48 rows of up to 6000 positions, 82 MB of pages to 291 MB of
// values, 62 us called again and again (6.0 TB/s; a copy reaches 5.1), 87 with the
// pages out of the caches (4.3); a page's heads by one workgroup 110 instead of
// 62.  A few rows: the sums and one turn, 7 us; 5875 tokens 10.
//
// Non-temporal stores: with cached ones those 48 rows take 91 us instead of 62.
// With a kernel that reads the values behind it, 900 positions 8.9 us and 8.7 with
// cached stores, 6000 22.0 and 21.6, 24000 48.3 and 45.8, 96000 213 and 224,
// 288000 637 and 653 (8 heads, fp16, both kernels).
#include "capi_util.h"
#include "kv4.h"
#include "rotary.h"

namespace oi2 {
namespace {

// kMostGroups: as many workgroups as are resident at a time, eight a CU, while
// their sums (12 bytes a row) leave room in LDS: up to 1700 rows or so.
constexpr int kThreads = 256, kWaves = kThreads / 64, kMostGroups = 2048;

struct FetchArgs {
  const int32_t *table, *lens, *first, *count;
  int32_t* cu;
  int n_seqs, width, max_len, n_pages, n_kv, max_tokens;
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
      __builtin_nontemporal_store(f32x4{z[0], z[1], z[2], z[3]}, reinterpret_cast<f32x4*>(p));
      __builtin_nontemporal_store(f32x4{z[4], z[5], z[6], z[7]}, reinterpret_cast<f32x4*>(p + 4));
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
      __builtin_nontemporal_store(u32x4{z[0], z[1], z[2], z[3]}, reinterpret_cast<u32x4*>(p));
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
__global__ __launch_bounds__(kThreads, 8) void k_kv4_fetch(FetchArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ uint2 s_wave[kWaves];
  const int n = a.n_seqs, tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // inclusive sums of the rows' tokens and of the pages that they lie in; the
  // first position of each row
  int32_t *s_tokens = lds, *s_pages = lds + n, *s_first = lds + 2 * n;
  const int per = (n + kThreads - 1) / kThreads, r0 = min(tid * per, n), r1 = min(r0 + per, n);
  uint2 mine = {0, 0};
  for (int r = r0; r < r1; ++r) {
    const int len = min(max(a.lens[r], 0), a.max_len), f = a.first ? min(max(a.first[r], 0), len) : 0;
    const int count = min(max(a.count[r], 0), len - f);
    mine.x = add_sat(mine.x, (uint32_t)count);
    mine.y = add_sat(mine.y, count ? (uint32_t)((f + count - 1) / kPage - f / kPage + 1) : 0);
    s_first[r] = f;
    s_tokens[r] = (int)mine.x;
    s_pages[r] = (int)mine.y;
  }
  uint2 upto = mine;                 // of the wave's lanes up to this one
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t x = (uint32_t)__shfl_up((int)upto.x, d), y = (uint32_t)__shfl_up((int)upto.y, d);
    if (lane >= d) upto = uint2{add_sat(upto.x, x), add_sat(upto.y, y)};
  }
  if (lane == 63) s_wave[wave] = upto;
  uint2 base = {(uint32_t)__shfl_up((int)upto.x, 1), (uint32_t)__shfl_up((int)upto.y, 1)};
  if (lane == 0) base = uint2{0, 0};
  __syncthreads();
  for (int w = 0; w < wave; ++w) base = uint2{add_sat(base.x, s_wave[w].x), add_sat(base.y, s_wave[w].y)};
  for (int r = r0; r < r1; ++r) {
    s_tokens[r] = (int)add_sat((uint32_t)s_tokens[r], base.x);
    s_pages[r] = (int)add_sat((uint32_t)s_pages[r], base.y);
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int r = tid; r <= n; r += kThreads) a.cu[r] = r ? s_tokens[r - 1] : 0;
  const int total = min(s_tokens[n - 1], a.max_tokens);

  // A wave has the places 4 wave + 16 k + i of a page, four at a time, whose
  // codes are 1 KB of k's and 1 KB of v's.
  const int u = lane & 15, i = lane >> 4, p0 = 4 * wave + i;
  const int k_at = k4_at(p0, u), v_at = v4_at(p0, u), ks_at = k4_scale_at(p0, u / 4), vs_at = v4_scale_at(p0, u / 4);
  auto row_where = [&](auto holds) {         // the first row that holds it
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (holds(mid)) hi = mid;
      else lo = mid + 1;
    }
    return __builtin_amdgcn_readfirstlane(lo);
  };
  int pages = s_pages[n - 1];
  if (s_tokens[n - 1] > total) {             // those up to the last token that fits
    const int r = row_where([&](int x) { return s_tokens[x] >= total; });
    const int left = total - (r ? s_tokens[r - 1] : 0), f = s_first[r];
    pages = (r ? s_pages[r - 1] : 0) + (left ? (f + left - 1) / kPage - f / kPage + 1 : 0);
  }
  const int64_t units = (int64_t)pages * a.n_kv;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int page = (int)(unit / a.n_kv), g = (int)(unit - (int64_t)page * a.n_kv);
    const int lo = row_where([&](int x) { return s_pages[x] > page; });
    const int t0 = lo ? s_tokens[lo - 1] : 0, t1 = min(s_tokens[lo], total);   // the row's tokens
    const int f = s_first[lo], j = f / kPage + page - (lo ? s_pages[lo - 1] : 0);
    int id = a.table[(int64_t)lo * a.width + j];
    id = (unsigned)id < (unsigned)a.n_pages ? id : 0;       // a damaged table reads page 0
    const rsrc_t b = rsrc(a.pages + ((int64_t)id * a.n_kv + g) * k4Block, k4Block);
    uint32_t kd[4], vd[4];
    uint16_t ks[4], vs[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {    // places 4 wave + 16 k + i
      kd[k] = bld4(b, k_at + 64 * k);
      vd[k] = bld4(b, v_at + 256 * k);
      ks[k] = bld2(b, ks_at + 32 * k);
      vs[k] = bld2(b, vs_at + 32 * k);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = (int64_t)t0 + j * kPage + p0 + 16 * k - f;
      if (t < t0 || t >= t1) continue;
      f16x2 y[4];
      values8(y, kd[k], ks[k]);
      store8<DTYPE>(a.dst[0], t * a.token_stride[0] + g * a.head_stride[0] + 8 * u, y, a.wide);
      values8(y, vd[k], vs[k]);
      store8<DTYPE>(a.dst[1], t * a.token_stride[1] + g * a.head_stride[1] + 8 * u, y, a.wide);
    }
  }

  if (a.zero) {
    const f16x2 none[4] = {};
    const int64_t rest = (int64_t)(a.max_tokens - total) * a.n_kv * 16;
    for (int64_t x = (int64_t)blockIdx.x * kThreads + tid; x < rest; x += (int64_t)gridDim.x * kThreads) {
      const int64_t t = total + x / (a.n_kv * 16);
      const int g = (int)(x / 16 % a.n_kv), w = (int)(x % 16);
#pragma unroll
      for (int e = 0; e < 2; ++e) store8<DTYPE>(a.dst[e], t * a.token_stride[e] + g * a.head_stride[e] + 8 * w, none, a.wide);
    }
  }
}

// Whether two different ones of (tokens, heads, 128) values share memory, or, with
// from != 0, one of them and one of the same values `from` elements further on:
// those dt tokens and dh heads apart are from + dt st + dh sh elements apart.
bool touch(int64_t tokens, int64_t heads, int64_t st, int64_t sh, int64_t from) {
  constexpr int64_t near = kHeadD - 1;
  for (int64_t dh = 1 - heads; dh < heads; ++dh) {
    const int64_t d = from + dh * sh;
    if (d >= -near && d <= near && (dh || from || (tokens > 1 && !st))) return true;
    if (tokens < 2 || !st) continue;
    // dt = 0 is done; the others nearest to -d / st
    int64_t dt = -d / st;
    dt = dt < 1 - tokens ? 1 - tokens : dt > tokens - 1 ? tokens - 1 : dt;
    for (int64_t x = dt - 1; x <= dt + 1; ++x)
      if (x && x > -tokens && x < tokens && d + x * st >= -near && d + x * st <= near) return true;
  }
  return false;
}

// Whether no two of the (tokens, heads, 128) values at h share memory.
bool apart(const oi2_heads* h, int64_t tokens) {
  const int64_t st = tokens > 1 ? h->token_stride : 0, sh = h->heads > 1 ? h->head_stride : 0, nh = h->heads;
  if (st < 0 || sh < 0) return false;
  // dense in either order: nothing to count
  if (sh >= kHeadD && st >= (nh - 1) * sh + kHeadD) return true;
  if (st >= kHeadD && sh >= (tokens - 1) * st + kHeadD) return true;
  return !touch(tokens, nh, st, sh, 0);
}

// Bytes from the first of them to the last one's end.
int64_t span(const oi2_heads* x, int64_t tokens, int size) {
  return ((tokens - 1) * x->token_stride + (x->heads - 1) * x->head_stride + kHeadD) * size;
}

// Whether those at k and at v do, or, with strides of their own, lie within one
// another's span.
bool meet(const oi2_heads* k, const oi2_heads* v, int64_t tokens, int size) {
  const int64_t t = tokens - 1, h = k->heads - 1;
  const uintptr_t a = (uintptr_t)k->data, b = (uintptr_t)v->data;
  if (a + span(k, tokens, size) <= b || b + span(v, tokens, size) <= a || a == b) return a == b;
  if ((t && k->token_stride != v->token_stride) || (h && k->head_stride != v->head_stride)) return true;
  return touch(tokens, k->heads, t ? k->token_stride : 0, h ? k->head_stride : 0, (int64_t)(b - a) / size);
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
  struct Range {
    const void* at;
    int64_t bytes;
  };
  auto cross = [](const Range& x, const Range& y) {
    const uintptr_t a = (uintptr_t)x.at, b = (uintptr_t)y.at;
    return a && b && a < b + y.bytes && b < a + x.bytes;
  };
  const int64_t rows = 4 * (int64_t)c->n_seqs, width = (c->max_len + kPage - 1) / kPage;
  const Range sums = {cu, rows + 4};
  const Range read[] = {{first, rows}, {count, rows}, {c->lens, rows}, {c->block_table, rows * width},
                        {c->pages, (int64_t)c->n_layers * c->n_pages * c->n_kv * k4Block}};
  for (const Range& r : read) OI2_CHECK_ARG(!cross(sums, r), "cu shares memory with what is read");
  for (const oi2_heads* x : {k, v}) {
    if (!max_tokens) break;
    const Range out = {x->data, span(x, max_tokens, dtype == OI2_DTYPE_F32 ? 4 : 2)};
    bool over = cross(out, sums);
    for (const Range& r : read) over = over || cross(out, r);
    OI2_CHECK_ARG(!over, "k or v shares memory with what is read, or with cu");
  }
  a.table = c->block_table;
  a.lens = c->lens;
  a.first = first;
  a.count = count;
  a.cu = cu;
  a.n_seqs = c->n_seqs;
  a.max_len = c->max_len;
  a.width = (int)width;
  a.n_pages = c->n_pages;
  a.n_kv = c->n_kv;
  a.max_tokens = max_tokens;
  a.zero = zero;
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * k4Block;
  // a page of one kv head is a workgroup's turn
  const int64_t some = c->n_seqs < max_tokens ? c->n_seqs : max_tokens, want = ((int64_t)max_tokens / kPage + 2 * some) * c->n_kv;
  const uint32_t groups = (uint32_t)(want < 1 ? 1 : want < kMostGroups ? want : kMostGroups);
  const size_t lds = (size_t)c->n_seqs * 12;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(groups), block(kThreads);
  if (dtype == OI2_DTYPE_F16) hipLaunchKernelGGL(k_kv4_fetch<OI2_DTYPE_F16>, grid, block, lds, st, a);
  else if (dtype == OI2_DTYPE_BF16) hipLaunchKernelGGL(k_kv4_fetch<OI2_DTYPE_BF16>, grid, block, lds, st, a);
  else hipLaunchKernelGGL(k_kv4_fetch<OI2_DTYPE_F32>, grid, block, lds, st, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}
