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
// (error <= 2^-25 half turns).  The frequencies come from the host as kernel parameters.
struct AppendArgs {
  PagedLayout kv;
  const float *k, *v, *q;
  float* q_out;
  void *kc, *vc;
  const uint32_t* start;
  size_t ks, vs, qs, qos;
  int heads, rows, rot;
  int* flags;
  double freq[128];  // base^(-2m / rot) / pi
};

// Sequence and position of row i; -1: none.  Raises the range flag where the page table does not
// hold the position.  Returns the element offset of the position for kv head 0.
__device__ bool append_slot(const AppendArgs& a, int i, int* pos, size_t* off) {
  const PagedLayout& kv = a.kv;
  int b = i;
  long long p;
  if (a.start) {
    if ((uint32_t)i < a.start[0] || (uint32_t)i >= a.start[kv.batch]) return false;
    int lo = 0, hi = kv.batch - 1;  // the last sequence with start[b] <= i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.start[mid] <= (uint32_t)i)
        lo = mid;
      else
        hi = mid - 1;
    }
    b = lo;
    if ((uint32_t)i >= a.start[b + 1]) return false;
    p = (long long)kv.lens[b] - a.start[b + 1] + i;
  } else {
    if (kv.lens[b] == 0) return false;
    p = (long long)kv.lens[b] - 1;
  }
  const long long page = p / kv.page_size;
  uint32_t id = 0xFFFFFFFFu;
  if (p >= 0 && page < kv.max_pages) id = kv.table[(size_t)b * kv.max_pages + page];
  if (id >= kv.n_pages) {
    atomicExch(&a.flags[FLAG_RANGE], RANGE_PAGE);
    return false;
  }
  *pos = (int)p;
  *off = (size_t)id * kv.page_stride + (size_t)(p - page * kv.page_size) * kv.slot_stride;
  return true;
}

// One block per row; VEC elements of one head per thread and step.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) k_paged_append(const __grid_constant__ AppendArgs a) {
  __shared__ float2 cs[128];
  __shared__ size_t s_off;
  __shared__ int s_pos, s_live;
  const int i = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x == 0) {
    int pos = 0;
    size_t off = 0;
    s_live = append_slot(a, i, &pos, &off);
    s_pos = pos;
    s_off = off;
  }
  __syncthreads();
  if (!s_live) return;
  for (int m = threadIdx.x; m < a.rot / 2; m += blockDim.x) {
    const double t = s_pos * a.freq[m];
    float sn, cn;
    sincospif((float)(t - 2.0 * rint(0.5 * t)), &sn, &cn);
    cs[m] = make_float2(cn, sn);
  }
  __syncthreads();
  const int per = a.kv.dim / VEC, heads = a.q ? a.heads : 0, kvh = a.kv.kv_heads;
  for (int e = threadIdx.x; e < (heads + 2 * kvh) * per; e += blockDim.x) {
    const int h = e / per, d = (e - h * per) * VEC;
    const float* src;
    float* qd = nullptr;
    T* cd = nullptr;
    bool turn = true;
    if (h < heads) {
      src = a.q + (size_t)i * a.qs + (size_t)h * a.kv.dim + d;
      qd = a.q_out + (size_t)i * a.qos + (size_t)h * a.kv.dim + d;
    } else if (h < heads + kvh) {
      src = a.k + (size_t)i * a.ks + (size_t)(h - heads) * a.kv.dim + d;
      cd = (T*)a.kc + s_off + (size_t)(h - heads) * a.kv.head_stride + d;
    } else {
      src = a.v + (size_t)i * a.vs + (size_t)(h - heads - kvh) * a.kv.dim + d;
      cd = (T*)a.vc + s_off + (size_t)(h - heads - kvh) * a.kv.head_stride + d;
      turn = false;
    }
    float x[VEC];
    if constexpr (VEC == 8) {
      *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(src);
      *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(src + 4);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) x[j] = src[j];
    }
    if (turn) {
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        if (d + j < a.rot) {
          const float2 r = cs[(d + j) >> 1];
          const float y0 = x[j] * r.x - x[j + 1] * r.y, y1 = x[j] * r.y + x[j + 1] * r.x;
          x[j] = y0;
          x[j + 1] = y1;
        }
      }
    }
    if (qd) {
      if constexpr (VEC == 8) {
        *reinterpret_cast<float4*>(qd) = *reinterpret_cast<float4*>(x);
        *reinterpret_cast<float4*>(qd + 4) = *reinterpret_cast<float4*>(x + 4);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) qd[j] = x[j];
      }
    } else {
      alignas(16) T y[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) y[j] = from_f32<T>(x[j]);
      if constexpr (VEC == 8) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(y) / 16; j++) reinterpret_cast<float4*>(cd)[j] = reinterpret_cast<float4*>(y)[j];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) cd[j] = y[j];
      }
    }
  }
}

template <typename T>
int append_launch(cudaStream_t st, const AppendArgs& a, bool vec) {
  TURT_CHECK_CUDA(launch_pdl(vec ? k_paged_append<T, 8> : k_paged_append<T, 2>, dim3(a.rows), dim3(256), 0, st, a));
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
  if (rot_dim && (ctx->rot_dim != rot_dim || ctx->rot_base != base)) {
    for (int m = 0; m < rot_dim / 2; m++) ctx->rot_freq[m] = pow((double)base, -2.0 * m / rot_dim) / M_PI;
    ctx->rot_dim = rot_dim;
    ctx->rot_base = base;
  }
  for (int m = 0; m < rot_dim / 2; m++) a.freq[m] = ctx->rot_freq[m];
  // 16-byte loads and stores: eight elements of a head per thread
  const size_t per = 16 / cache_type_size(kv->dtype);
  const bool vec = kv->head_dim % 8 == 0 && aligned16(k) && aligned16(v) && k_stride % 4 == 0 && v_stride % 4 == 0 &&
                   (!q || (aligned16(q) && aligned16(q_out) && q_stride % 4 == 0 && q_out_stride % 4 == 0)) &&
                   aligned16(kv->k) && aligned16(kv->v) && a.kv.page_stride % per == 0 && a.kv.head_stride % per == 0 &&
                   a.kv.slot_stride % per == 0;
  if (kv->dtype == TURT_CACHE_F32) return append_launch<float>(ctx->stream, a, vec);
  if (kv->dtype == TURT_CACHE_F16) return append_launch<__half>(ctx->stream, a, vec);
  return append_launch<__nv_bfloat16>(ctx->stream, a, vec);
}
