// paged.cu -- the paged key / value cache: its descriptor, and appending new positions with their
// rotation (reading it: paged_attend.cu).
//
// The single-sequence decode step (decode.cu) keeps one contiguous fp32 cache with as many key
// heads as query heads.  Here many sequences share a pool of pages (so none reserves its longest
// length), several query heads may read one key head, and the cache may be stored in 16 bits;
// activations stay fp32, as everywhere in this library.
#include <math.h>

#include "ctx.cuh"
#include "paged.cuh"

namespace turt {

int paged_layout(const turt_paged_kv* kv, PagedLayout* out) {
  TURT_REQUIRE(kv, "paged cache: null descriptor");
  TURT_REQUIRE(kv->dtype == TURT_CACHE_F32 || kv->dtype == TURT_CACHE_F16 || kv->dtype == TURT_CACHE_BF16,
               "paged cache: type must be TURT_CACHE_F32, TURT_CACHE_F16 or TURT_CACHE_BF16");
  TURT_REQUIRE(kv->batch >= 0, "paged cache: negative batch");
  TURT_REQUIRE(kv->n_pages > 0 && kv->page_size > 0 && kv->n_kv_head > 0 && kv->max_pages > 0,
               "paged cache: pages, page size, heads and table width must be positive");
  TURT_REQUIRE(kv->head_dim >= 2 && kv->head_dim <= 256 && kv->head_dim % 2 == 0,
               "paged cache: head_dim must be even, 2 .. 256");
  TURT_REQUIRE((long long)kv->max_pages * kv->page_size <= 0x7fffffffLL,
               "paged cache: max_pages * page_size must be below 2^31");
  TURT_REQUIRE(kv->k && kv->v && kv->page_table && kv->lens, "paged cache: null pointer");
  const uintptr_t size = cache_type_size(kv->dtype);
  TURT_REQUIRE((uintptr_t)kv->k % size == 0 && (uintptr_t)kv->v % size == 0 && (uintptr_t)kv->page_table % 4 == 0 &&
                   (uintptr_t)kv->lens % 4 == 0,
               "paged cache: misaligned pointer");
  const size_t d = kv->head_dim;
  PagedLayout p;
  if (!kv->page_stride && !kv->head_stride && !kv->slot_stride) {
    p.slot_stride = d;
    p.head_stride = d * kv->page_size;
    p.page_stride = p.head_stride * kv->n_kv_head;
  } else {
    p.slot_stride = kv->slot_stride;
    p.head_stride = kv->head_stride;
    p.page_stride = kv->page_stride;
    const size_t far = (size_t)1 << 40;
    TURT_REQUIRE(p.slot_stride <= far && p.head_stride <= far && p.page_stride <= far, "paged cache: stride too large");
    TURT_REQUIRE((kv->page_size == 1 || p.slot_stride >= d) && (kv->n_kv_head == 1 || p.head_stride >= d) &&
                     (kv->n_pages == 1 || p.page_stride >= d),
                 "paged cache: strides let positions overlap");
  }
  // strides of single entries are never used: legal values
  if (kv->page_size == 1) p.slot_stride = d;
  if (kv->n_kv_head == 1) p.head_stride = p.slot_stride;
  if (kv->n_pages == 1) p.page_stride = p.slot_stride;
  p.table = kv->page_table;
  p.lens = kv->lens;
  p.n_pages = kv->n_pages;
  p.page_size = kv->page_size;
  p.max_pages = kv->max_pages;
  p.kv_heads = kv->n_kv_head;
  p.dim = (int)d;
  p.batch = kv->batch;
  *out = p;
  return OK;
}

namespace {

// --------------------------------------------------------------------------------- append
//
//   y[2m] = x[2m] cos a - x[2m+1] sin a,  y[2m+1] = x[2m] sin a + x[2m+1] cos a,
//   a = position * base^(-2m / rot)
// A position of 10^5 and more leaves an fp32 product a with an error of whole hundredths of a
// turn, so a / pi is formed and reduced to [-1, 1] in double and only then rounded for sincospif
// (error <= 2^-25 half turns).  Bound by the memory traffic where rows are many and by the chain
// start -> page table -> store where they are few: a thread asks for its elements before it knows
// where they go, and a warp looks up one row, 32 entries of `start` at a time.
struct AppendArgs {
  PagedLayout kv;
  const float *k, *v, *q;
  float* q_out;
  void *kc, *vc;
  const uint32_t* start;
  size_t ks, vs, qs, qos;
  int heads, rows, rot;
  int per_block;       // rows per block
  uint32_t items;      // pieces of VEC elements per row
  uint64_t row_mul;    // e / items = e * row_mul >> 32 (several rows per block: e < 2^13)
  uint64_t head_mul;   // e / (dim / VEC) likewise (e < 2^25)
  double step;         // 2 log2(base) / rot
  int* flags;
};

constexpr int kAppendThreads = 256, kAppendRows = 8;

// One warp: sequence and position of row i; false where it has none.  Raises the range flag where the
// page table does not hold the position.  off: the element offset of the position for kv head 0.
__device__ bool append_slot(const AppendArgs& a, int i, int lane, int* pos, size_t* off) {
  const PagedLayout& kv = a.kv;
  int b = i;
  long long p;
  if (a.start) {
    // the last sequence with start[b] <= i, in steps of a 32nd of what is left
    int lo = 0, n = kv.batch;  // it is among lo .. lo + n - 1, or there is none
    while (n > 1) {
      const int piece = (n + 31) / 32, x = lo + lane * piece;
      const uint32_t in = __ballot_sync(0xffffffffu, x < lo + n && a.start[x] <= (uint32_t)i);
      if (in == 0) return false;
      const int to = lo + (31 - __clz(in)) * piece;
      n = min(piece, lo + n - to);
      lo = to;
    }
    b = lo;
    const uint32_t first = a.start[b], next = a.start[b + 1];
    if ((uint32_t)i < first || (uint32_t)i >= next) return false;
    p = (long long)kv.lens[b] - next + i;
  } else {
    if (kv.lens[b] == 0) return false;
    p = (long long)kv.lens[b] - 1;
  }
  uint32_t id = 0xFFFFFFFFu;
  const uint32_t page = (uint32_t)p / kv.page_size;
  if (p >= 0 && page < kv.max_pages) id = kv.table[(size_t)b * kv.max_pages + page];
  if (id >= kv.n_pages) {
    if (lane == 0) atomicExch(&a.flags[FLAG_RANGE], RANGE_PAGE);
    return false;
  }
  *pos = (int)p;
  *off = (size_t)id * kv.page_stride + (size_t)((uint32_t)p - page * kv.page_size) * kv.slot_stride;
  return true;
}

template <int VEC>
struct AppendPiece {
  const float* src;
  int r, h, d;  // row of the block, head (queries, keys, values), first element
  float x[VEC];
};

template <int VEC>
__device__ __forceinline__ void append_load(const AppendArgs& a, uint32_t e, int row0, AppendPiece<VEC>& p) {
  const int heads = a.q ? a.heads : 0, kvh = a.kv.kv_heads, dim = a.kv.dim;
  p.r = a.per_block > 1 ? (int)(e * a.row_mul >> 32) : 0;
  const uint32_t in = e - p.r * a.items;
  p.h = (int)(in * a.head_mul >> 32);
  p.d = (int)(in - p.h * (dim / VEC)) * VEC;
  const size_t i = row0 + p.r;
  if (p.h < heads)
    p.src = a.q + i * a.qs + (size_t)p.h * dim;
  else if (p.h < heads + kvh)
    p.src = a.k + i * a.ks + (size_t)(p.h - heads) * dim;
  else
    p.src = a.v + i * a.vs + (size_t)(p.h - heads - kvh) * dim;
  p.src += p.d;
  if constexpr (VEC == 8) {
    *reinterpret_cast<float4*>(p.x) = *reinterpret_cast<const float4*>(p.src);
    *reinterpret_cast<float4*>(p.x + 4) = *reinterpret_cast<const float4*>(p.src + 4);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) p.x[j] = p.src[j];
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void append_store(const AppendArgs& a, int row0, const float2* cs, size_t off, AppendPiece<VEC>& p) {
  const int heads = a.q ? a.heads : 0, kvh = a.kv.kv_heads;
  if (p.h < heads + kvh) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      if (p.d + j < a.rot) {
        const float2 r = cs[(p.d + j) >> 1];
        const float y0 = p.x[j] * r.x - p.x[j + 1] * r.y, y1 = p.x[j] * r.y + p.x[j + 1] * r.x;
        p.x[j] = y0;
        p.x[j + 1] = y1;
      }
    }
  }
  if (p.h < heads) {
    float* to = a.q_out + (size_t)(row0 + p.r) * a.qos + (size_t)p.h * a.kv.dim + p.d;
    if constexpr (VEC == 8) {
      *reinterpret_cast<float4*>(to) = *reinterpret_cast<float4*>(p.x);
      *reinterpret_cast<float4*>(to + 4) = *reinterpret_cast<float4*>(p.x + 4);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) to[j] = p.x[j];
    }
    return;
  }
  const bool key = p.h < heads + kvh;
  T* to = (T*)(key ? a.kc : a.vc) + off + (size_t)(p.h - heads - (key ? 0 : kvh)) * a.kv.head_stride + p.d;
  alignas(16) T y[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) y[j] = from_f32<T>(p.x[j]);
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(y) / 16; j++) reinterpret_cast<float4*>(to)[j] = reinterpret_cast<float4*>(y)[j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) to[j] = y[j];
  }
}

// per_block rows per block; VEC elements of one head per thread and piece.  Resident threads count for
// more than pieces under way per thread: eight blocks per SM with one piece each measured 47.5 us for
// 6318 rows of 48 heads of 128 (285 MB), four blocks with four pieces 55 us.
template <typename T, int VEC>
__global__ void __launch_bounds__(kAppendThreads, 8) k_paged_append(const __grid_constant__ AppendArgs a) {
  __shared__ float2 cs[kAppendRows][128];
  __shared__ size_t s_off[kAppendRows];
  __shared__ int s_pos[kAppendRows];  // -1: the row goes nowhere
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int row0 = blockIdx.x * a.per_block, n = min(a.per_block, a.rows - row0);
  const int half = a.rot >> 1;
  double freq = 0.0;  // base^(-2m / rot) / pi of pair m = tid % half
  const int m = half ? tid % half : 0;
  if (half) freq = exp2(-a.step * m) * 0.31830988618379067;
  pdl_wait();
  pdl_trigger();
  AppendPiece<VEC> p;
  const uint32_t total = n * a.items;
  if (tid < total) append_load<VEC>(a, tid, row0, p);
  if (w < n) {
    int pos = -1;
    size_t off = 0;
    if (!append_slot(a, row0 + w, lane, &pos, &off)) pos = -1;
    if (lane == 0) {
      s_pos[w] = pos;
      s_off[w] = off;
    }
  }
  __syncthreads();
  if (half) {
    // a thread keeps its pair and goes through the rows
    const int lanes = kAppendThreads / half, r0 = tid / half;
    if (r0 < lanes)
      for (int r = r0; r < n; r += lanes) {
        const double t = s_pos[r] * freq;
        float sn, cn;
        sincospif((float)(t - 2.0 * rint(0.5 * t)), &sn, &cn);
        cs[r][m] = make_float2(cn, sn);
      }
    __syncthreads();
  }
  for (uint32_t e = tid; e < total; e += kAppendThreads) {
    if (s_pos[p.r] >= 0) append_store<T, VEC>(a, row0, cs[p.r], s_off[p.r], p);
    if (e + kAppendThreads < total) append_load<VEC>(a, e + kAppendThreads, row0, p);
  }
}

template <typename T, int VEC>
int append_launch(cudaStream_t st, AppendArgs a) {
  a.items = (uint32_t)(((a.q ? a.heads : 0) + 2 * a.kv.kv_heads) * (a.kv.dim / VEC));
  // up to six pieces per thread, as long as there are two blocks per SM: 4543 rows of 25 heads of 80
  // took 18.1 us one to a block, 14.8 two, 14.3 four, 16.4 eight
  int per = 1;
  while (per < kAppendRows && 2 * per * a.items <= 6 * kAppendThreads && a.rows / (2 * per) >= 2 * 148) per *= 2;
  a.per_block = per;
  auto mul = [](uint32_t d) { return ((1ull << 32) + d - 1) / d; };
  a.row_mul = mul(a.items);
  a.head_mul = mul(a.kv.dim / VEC);
  TURT_CHECK_CUDA(launch_pdl(k_paged_append<T, VEC>, dim3(ceil_div(a.rows, per)), dim3(kAppendThreads), 0, st, a));
  TURT_LAUNCH_CHECK();
  return OK;
}

}  // namespace
}  // namespace turt

using namespace turt;

extern "C" int turt_paged_append(turt_ctx* ctx, const turt_paged_kv* kv, const float* k, size_t k_stride,
                                 const float* v, size_t v_stride, const float* q, size_t q_stride, float* q_out,
                                 size_t q_out_stride, int n_head, const uint32_t* start, int rows, int rot_dim,
                                 float base) {
  AppendArgs a;
  RC(paged_layout(kv, &a.kv));
  TURT_REQUIRE(rows >= 0, "paged_append: negative rows");
  TURT_REQUIRE(start || rows == kv->batch, "paged_append: without start there is one row per sequence");
  TURT_REQUIRE(rot_dim >= 0 && rot_dim <= kv->head_dim && rot_dim % 2 == 0,
               "paged_append: rot_dim must be even, 0 .. head_dim");
  TURT_REQUIRE(rot_dim == 0 || (base > 0.0f && isfinite(base)), "paged_append: base must be positive");
  const size_t wide = (size_t)kv->n_kv_head * kv->head_dim;
  TURT_REQUIRE(rows == 0 || (k && v), "paged_append: null pointer");
  TURT_REQUIRE(rows <= 1 || (k_stride >= wide && v_stride >= wide), "paged_append: row strides below the row width");
  if (q) {
    TURT_REQUIRE(n_head > 0 && q_out, "paged_append: queries need heads and an output");
    TURT_REQUIRE(rows <= 1 || (q_stride >= (size_t)n_head * kv->head_dim && q_out_stride >= (size_t)n_head * kv->head_dim),
                 "paged_append: query strides below the row width");
    TURT_REQUIRE(q_out != q || q_stride == q_out_stride, "paged_append: rotating in place needs equal strides");
  }
  TURT_REQUIRE(((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)start) % 4 == 0,
               "paged_append: misaligned pointer");
  TURT_REQUIRE(ctx, "null context");
  TURT_CHECK_CUDA(cudaSetDevice(ctx->device));
  if (rows == 0 || kv->batch == 0) return OK;
  a.k = k, a.v = v, a.q = q, a.q_out = q_out;
  a.kc = kv->k, a.vc = kv->v;
  a.start = start;
  a.ks = k_stride, a.vs = v_stride, a.qs = q_stride, a.qos = q_out_stride;
  a.heads = n_head, a.rows = rows, a.rot = rot_dim;
  a.flags = ctx->flags;
  a.step = rot_dim ? 2.0 * log2((double)base) / rot_dim : 0.0;
  // 16-byte loads and stores: eight elements of a head per thread
  const size_t per = 16 / cache_type_size(kv->dtype);
  const bool vec = kv->head_dim % 8 == 0 && aligned16(k) && aligned16(v) && k_stride % 4 == 0 && v_stride % 4 == 0 &&
                   (!q || (aligned16(q) && aligned16(q_out) && q_stride % 4 == 0 && q_out_stride % 4 == 0)) &&
                   aligned16(kv->k) && aligned16(kv->v) && a.kv.page_stride % per == 0 && a.kv.head_stride % per == 0 &&
                   a.kv.slot_stride % per == 0;
  if (kv->dtype == TURT_CACHE_F32) return vec ? append_launch<float, 8>(ctx->stream, a) : append_launch<float, 2>(ctx->stream, a);
  if (kv->dtype == TURT_CACHE_F16)
    return vec ? append_launch<__half, 8>(ctx->stream, a) : append_launch<__half, 2>(ctx->stream, a);
  return vec ? append_launch<__nv_bfloat16, 8>(ctx->stream, a) : append_launch<__nv_bfloat16, 2>(ctx->stream, a);
}
