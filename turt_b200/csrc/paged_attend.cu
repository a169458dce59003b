// paged_attend.cu -- attention of one new token per sequence over a paged key / value cache.
//
//   s_j = scale q . k_j,  out = sum_j 2^(s_j' - m) v_j / sum_j 2^(s_j' - m),  s' = s log2(e)
//
// Every cached key and value is used by the heads of its group only and read once for eight of them
// (for four where heads have more than 128 elements), so the bound is the memory bandwidth.  The
// positions of all sequences and key heads form one line of tiles, cut into equal stretches, one per
// warp of a grid that fills the GPU once: ragged lengths, one long sequence and many short ones load
// all warps alike, whatever the lengths are (they are read on the device).  A warp streams its tiles
// through a ring of shared memory of its own, filled by bulk tensor copies that one lane issues, so
// nothing but its own copies holds it up; it runs the online softmax of its stretch in registers.  A
// part of a sequence that a warp did not see whole is joined with its neighbours': first inside the
// block, then by the last block to arrive, always in the order of positions.
//
// Measured on a B200 (changing inputs): 96 sequences of up to 8192, 32 query / 8 key heads of 128, bf16
// (1.63 GB): 260 us, 6.3 TB/s; one of 131001 (537 MB): 93 us, 5.7 TB/s; 64 of up to 1024, 12 heads of
// 64, fp32 (204 MB): 41 us, 5.0 TB/s.  Of the last, about 5 us pass before the first tile has arrived
// (length -> page table -> copy, each a trip to memory) and 4 us in the joins.
#include <math.h>

#include <algorithm>

#include "ctx.cuh"
#include "gemm.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace turt {
namespace {

constexpr int kMaxBlocks = 512;           // counters and partial results in the workspace
constexpr int kPrefix = 1024;             // entries of the tile prefix held in shared memory
constexpr int kGroup = 8;                 // heads of a group that a warp treats at once, at most
// What a sequence part costs besides its tiles, in tiles: 1000 sequences of 1 .. 300 positions, 16 / 8 bf16
// heads of 64, took 98 / 78 / 69 / 71 us at 0 / 1 / 2 / 3.
constexpr int kPartCost = 2;
constexpr float kLazy = 8.0f;             // the running max moves when it is this far behind (log2)
constexpr int kWaitSite = 40;             // reported when a copy's wait runs out

struct AttendArgs {
  PagedLayout kv;
  const void *kc, *vc;
  const float* q;
  float *out, *lse;
  size_t qs, os;
  int heads, group, window;
  int chunks;        // parts of a group: ceil(group / heads per part)
  int part;          // heads per part
  float scale;       // times log2(e)
  uint32_t div_mul;  // position / page_size = position * div_mul >> div_shift (positions < 2^31)
  int div_shift;
  int min_tiles;     // tiles per warp, at least
  int whole_tiles;   // tiles per warp up to which a block takes whole sequence parts
  int box_rows;      // positions per copy
  int page_tiles;    // tiles per page where tiles do not cross pages, 0: any KT positions are a tile
  uint32_t* counters;
  float* partial;
  int* flags;
  int dtype;
  bool q_pairs;  // the elements of q can be read two at a time
};

__device__ __forceinline__ uint32_t page_of(const AttendArgs& a, uint32_t j) {
  return (uint32_t)(((uint64_t)j * a.div_mul) >> a.div_shift);
}

__device__ __forceinline__ float exp2_of(float s, float m) { return exp2f(s - (m == -INFINITY ? 0.f : m)); }

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ unsigned add_acq_rel(uint32_t* p) {
  unsigned old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
  return old;
}

__device__ __forceinline__ unsigned long long div64(unsigned long long x, unsigned long long y) {
  return (x | y) >> 32 ? x / y : (unsigned)x / (unsigned)y;
}

// The positions that sequence b attends to: [first, n) in tiles [t0, t1).  A tile is KT positions, or,
// where KT (in pieces of box_rows) does not divide the page size, KT slots of one page.
struct Seq {
  uint32_t n, first, t0, t1;
};
template <int KT>
__device__ __forceinline__ uint32_t tile_of(const AttendArgs& a, uint32_t j) {
  if (!a.page_tiles) return j / KT;
  const uint32_t pg = page_of(a, j);
  return pg * a.page_tiles + (j - pg * a.kv.page_size) / KT;
}
// Positions [j0, j1) of tile t.
template <int KT>
__device__ __forceinline__ void tile_span(const AttendArgs& a, uint32_t t, uint32_t* j0, uint32_t* j1) {
  if (!a.page_tiles) {
    *j0 = t * KT;
    *j1 = *j0 + KT;
  } else {
    const uint32_t pg = t / a.page_tiles;
    *j0 = pg * a.kv.page_size + (t - pg * a.page_tiles) * KT;
    *j1 = min(*j0 + KT, (pg + 1) * a.kv.page_size);
  }
}
template <int KT>
__device__ __forceinline__ Seq seq_of(const AttendArgs& a, int b) {
  Seq s;
  s.n = a.kv.lens[b];
  if (s.n > a.kv.max_pages * a.kv.page_size) s.n = 0;  // flagged where the batch is scanned
  s.first = a.window > 0 && s.n > (uint32_t)a.window ? s.n - a.window : 0;
  s.t0 = s.t1 = 0;
  if (s.n) {
    s.t0 = tile_of<KT>(a, s.first);
    s.t1 = tile_of<KT>(a, s.n - 1) + 1;
  }
  return s;
}

// A place on the line: sequence, part of a head group, tile.  On the line a sequence part takes up
// kPartCost places and then one per tile, so that a warp with many short parts gets fewer tiles.
template <int KT>
struct Walk {
  Seq s;
  int b, hc;
  uint32_t t;
  unsigned long long pos;
  __device__ void next(const AttendArgs& a, int hcs) {
    pos++;
    if (++t < s.t1) return;
    pos += kPartCost;
    t = s.t0;
    if (++hc < hcs) return;
    hc = 0;
    do {
      if (++b >= a.kv.batch) return;
      s = seq_of<KT>(a, b);
    } while (s.n == 0);
    t = s.t0;
  }
};

// A result of part of a sequence: per head m (log2), l and dim unnormalised outputs.  Two 16-byte units
// at least: the join divides by the number of units through a 32-bit reciprocal, which 1 has none of.
__host__ __device__ __forceinline__ int rec_floats(int part, int dim) {
  const int n = (part * (dim + 2) + 3) & ~3;
  return n < 8 ? 8 : n;
}

__device__ __forceinline__ float weight_of(float m, float l, float top) {
  return m == -INFINITY && l == 0.f ? 0.f : exp2f(m - top);
}

// The heads of part hc of the head groups: kv head, first query head, how many.
struct HeadPart {
  int kv, head, n;
};
__device__ __forceinline__ HeadPart head_part(const AttendArgs& a, int hc) {
  int kv = hc, g0 = 0;
  if (a.chunks > 1) {
    kv = hc / a.chunks;
    g0 = (hc - kv * a.chunks) * a.part;
  }
  return {kv, kv * a.group + g0, min(a.part, a.group - g0)};
}

__device__ __forceinline__ void store_out(const AttendArgs& a, int b, int head, int d, float o, float l) {
  a.out[(size_t)b * a.os + (size_t)head * a.kv.dim + d] = l == 0.f ? 0.f : o / l;
}
__device__ __forceinline__ void store_lse(const AttendArgs& a, int b, int head, float m, float l) {
  if (a.lse) a.lse[(size_t)b * a.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// One head's outputs, element lane + 32 k in o[k].
__device__ __forceinline__ void store_head(const AttendArgs& a, int b, int head, int lane, const float (&o)[8], float m, float l) {
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (lane + 32 * k < a.kv.dim) store_out(a, b, head, lane + 32 * k, o[k], l);
  if (lane == 0) store_lse(a, b, head, m, l);
}

// One warp, any layout: positions [j0, j1) of sequence b into rec (one record of a.part heads), four
// positions and GH heads at a time.  Lanes take every 32nd element, NI of them.  The formula as it
// stands: also what a stretch with infinities or NaN falls back to.
template <typename T, int NI, int GH>
__device__ __noinline__ void attend_plain(const AttendArgs& a, int b, int hc, uint32_t j0, uint32_t j1, float* rec) {
  constexpr int AT_ONCE = 4;
  const PagedLayout& kv = a.kv;
  const int lane = threadIdx.x & 31, dim = kv.dim;
  const HeadPart hp = head_part(a, hc);
  for (int g0 = 0; g0 < a.part; g0 += GH) {
    float q[GH][NI], o[GH][NI], m[GH], l[GH];
#pragma unroll
    for (int g = 0; g < GH; g++) {
      const bool head = g0 + g < hp.n;
      const float* qh = a.q + (size_t)b * a.qs + (size_t)(hp.head + (head ? g0 + g : 0)) * dim;
#pragma unroll
      for (int i = 0; i < NI; i++) {
        q[g][i] = head && lane + 32 * i < dim ? qh[lane + 32 * i] * a.scale : 0.f;
        o[g][i] = 0.f;
      }
      m[g] = -INFINITY;
      l[g] = 0.f;
    }
    for (uint32_t j = j0; j < j1; j += AT_ONCE) {
      // lanes 0 .. AT_ONCE - 1 look up a position each
      size_t off = 0;
      bool there = false;
      if (lane < AT_ONCE && j + lane < j1) {
        const uint32_t pg = page_of(a, j + lane), id = kv.table[(size_t)b * kv.max_pages + pg];
        there = id < kv.n_pages;
        if (!there)
          atomicExch(&a.flags[FLAG_RANGE], RANGE_PAGE);
        else
          off = (size_t)id * kv.page_stride + (size_t)hp.kv * kv.head_stride +
                (size_t)(j + lane - pg * kv.page_size) * kv.slot_stride;
      }
      const uint32_t live = __ballot_sync(0xffffffffu, there);
      float k[AT_ONCE][NI], v[AT_ONCE][NI];
#pragma unroll
      for (int x = 0; x < AT_ONCE; x++) {
        const size_t at = __shfl_sync(0xffffffffu, off, x);  // position 0 of the cache where there is none
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const bool in = lane + 32 * i < dim;
          k[x][i] = in ? to_f32(((const T*)a.kc)[at + lane + 32 * i]) : 0.f;
          v[x][i] = in ? to_f32(((const T*)a.vc)[at + lane + 32 * i]) : 0.f;
        }
      }
#pragma unroll
      for (int g = 0; g < GH; g++) {
        float s[AT_ONCE], top = m[g];
#pragma unroll
        for (int x = 0; x < AT_ONCE; x++) {
          s[x] = 0.f;
#pragma unroll
          for (int i = 0; i < NI; i++)
            if (lane + 32 * i < dim) s[x] += q[g][i] * k[x][i];
          s[x] = warp_sum(s[x]);
          if (!((live >> x) & 1)) s[x] = -INFINITY;
          top = fmaxf(top, s[x]);
        }
        const float f = top == -INFINITY ? 1.f : exp2f(m[g] - top);
        m[g] = top;
        l[g] *= f;
#pragma unroll
        for (int i = 0; i < NI; i++) o[g][i] *= f;
#pragma unroll
        for (int x = 0; x < AT_ONCE; x++) {
          if (s[x] == -INFINITY) continue;  // no weight, whatever the value is
          const float p = exp2f(s[x] - top);
          l[g] += p;
#pragma unroll
          for (int i = 0; i < NI; i++) o[g][i] += p * v[x][i];
        }
      }
    }
#pragma unroll
    for (int g = 0; g < GH; g++) {
      if (g0 + g >= a.part) continue;
      float* r = rec + (g0 + g) * (dim + 2);
      if (lane == 0) {
        r[0] = m[g];
        r[1] = l[g];
      }
#pragma unroll
      for (int i = 0; i < NI; i++)
        if (lane + 32 * i < dim) r[2 + lane + 32 * i] = o[g][i];
    }
  }
  __syncwarp();
}
// The running maximum may lie up to kLazy behind, with weights above 1.  Where sums are so large that the joins
// could take them out of range, they are brought to weights of 1 at most, as the exact maximum gives.  Returns
// whether there were such sums, or any that are not finite (the same for the warp).
template <int N, int K>
__device__ __forceinline__ bool below_one(float (&acc)[N][K], float& m, float& l) {
  bool big = !(fabsf(l) <= 0x1p100f);
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int k = 0; k < K; k++) big |= !(fabsf(acc[i][k]) <= 0x1p100f);
  if (!__any_sync(0xffffffffu, big)) return false;
  constexpr float down = 1.f / (1 << (int)kLazy);
  m += kLazy;
  l *= down;
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int k = 0; k < K; k++) acc[i][k] *= down;
  return true;
}
template <int N, int K>
__device__ __forceinline__ bool all_finite(const float (&acc)[N][K], float l) {
  bool bad = !(fabsf(l) < INFINITY);
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int k = 0; k < K; k++) bad |= !(fabsf(acc[i][k]) < INFINITY);
  return !__any_sync(0xffffffffu, bad);
}

// Paths: how a warp treats the tiles of its stretch.
//   begin / tile / finish   the softmax of one part of a sequence; finish leaves its record in rec, or
//                           returns false where something in it is not finite
//   A tile lies in its stage of the ring as KT rows of keys and then KT of values, in slabs of SLAB
//   elements (a slab holds all KT rows); `ok` has a bit for each row that is attended to, and the
//   value rows without one are zero.
// ------------------------------------------------------------------------------- any layout
template <typename T>
struct PathPlain {  // attend_plain alone
  using Type = T;
  static constexpr int KT = 16, WARPS = 8, STAGES = 1, STAGE_BYTES = 0, BLOCKS = 2, MAX_DIM = 256;
  static constexpr bool RING = false;
};

// -------------------------------------------------------------- 16-bit caches: tensor cores
//
// A tile is 16 or 32 positions.  S = Q K^T and O += P V are m16n8k16 products with the heads of the group
// (8 at most) as rows.  Only the cache is 16-bit: q and the weights p are fp32 and go in as a sum of
// 16-bit parts, one part in rows 0-7 and the next in rows 8-15 of the same product, so the unused
// half of the rows buys the precision.  bf16 takes three parts (24 bits): up to four heads have the second
// in rows 4-7 and the third in rows 8-11, more heads the third in a product of its own.  fp16 takes two:
// what the first leaves is at most 2^-11 of the element and goes in multiplied by 2^11, so that it is not
// lost among fp16's subnormals, and its products come back times 2^-11 in fp32.  Both roundings are to 11
// bits and signed, which leaves an error of 2^-23 of the element, as long as it is not among the
// subnormals itself: q is scaled per head by a power of two to a maximum in [2^14, 2^15), so an element is off
// by 2^-23 of itself or 2^-50 of the largest.  The weights of a tile are scaled per head in the same way, to a
// maximum in (2^13, 2^14], and the tile's product and sum come back times a power of two when they are added to the
// running ones: a weight is off by 2^-23 of itself or 2^-49 of its tile's largest, however small that is next
// to the sequence's.  The thread that holds row r also holds
// row r + 8 (and the one 16 lanes on row r + 4), so the parts of a score meet after a shuffle at most,
// and the scores are where the next product wants p.  Each tile's product is added to the running
// output in fp32 outside the tensor cores, whose own accumulation truncates.
// Infinities and NaN break the parts (0 * inf).
template <typename T>
struct Half2;
template <>
struct Half2<__half> {
  static constexpr bool THREE = false;
  static constexpr float UP = 2048.f, DOWN = 1.f / 2048.f;  // the second part's scale
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                             const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};
template <>
struct Half2<__nv_bfloat16> {
  static constexpr bool THREE = true;
  static constexpr float UP = 1.f, DOWN = 1.f;
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                             const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// KD: steps of 16 elements that cover head_dim (a multiple of 8).  QUAD: at most four heads.
template <typename T, int KD, bool QUAD>
struct PathMma {
  using Type = T;
  using H = Half2<T>;
  // heads of up to 64 elements: twice the positions, for the work per tile that does not grow with them
  // (16 / 8 heads of 64, 32 x 4000 positions: 49 us; with tiles of 16 positions it was 66, and 50)
  static constexpr int KT = KD <= 4 ? 32 : 16, WARPS = 8, NB = KT / 8;
  static constexpr int MAX_DIM = KD * 16;
  static constexpr bool RING = true;
  static constexpr bool SPLIT = QUAD && H::THREE;    // parts in rows r, r + 4, r + 8
  static constexpr bool EXTRA = !QUAD && H::THREE;   // a product for the third part
  // slabs of KT rows of 128 (64) bytes whose 16-byte units are exchanged (unit ^ row % 8, unit ^ row / 2 % 4):
  // the eight rows of an ldmatrix fall into different banks
  static constexpr int SLAB = KD <= 2 ? 32 : 64, SLABS = (KD + 3) / 4, ROW = SLAB * 2, SLAB_BYTES = KT * ROW;
  static constexpr int SWIZZLE = ROW;
  static constexpr int STAGE_BYTES = 2 * SLABS * SLAB_BYTES;
  static constexpr int STAGES = 2, BLOCKS = KD <= 2 ? 2 : 1;  // BLOCKS: resident per SM

  uint32_t qa[KD][4], qb[EXTRA ? KD : 1][2];
  float acc[2 * KD][2], m, l, unscale;

  // The parts of (u, v) for rows r and r + 8 of a product, and the third part's own.
  static __device__ __forceinline__ void parts(float u, float v, uint32_t& x, uint32_t& y, uint32_t& z) {
    const uint32_t p0 = H::pack(u, v);
    const float2 f0 = H::unpack(p0);
    u = (u - f0.x) * H::UP, v = (v - f0.y) * H::UP;
    const uint32_t p1 = H::pack(u, v);
    x = p0, y = p1;
    if constexpr (H::THREE) {
      const float2 f1 = H::unpack(p1);
      const uint32_t p2 = H::pack(u - f1.x, v - f1.y);
      if constexpr (SPLIT) {
        const bool second = (threadIdx.x & 16) != 0;
        x = second ? p1 : p0;
        y = second ? 0u : p2;
      }
      z = p2;
    }
  }

  __device__ static int row() { return SPLIT ? (threadIdx.x & 15) >> 2 : (threadIdx.x & 31) >> 2; }

  __device__ void begin(const AttendArgs& a, int b, int hc) {
    const int r = row(), c = (threadIdx.x & 3) * 2, dim = a.kv.dim;
    const HeadPart hp = head_part(a, hc);
    const float* q = a.q + (size_t)b * a.qs + (size_t)(hp.head + (r < hp.n ? r : 0)) * dim + c;
    float x[KD][4], top = 0.f;
#pragma unroll
    for (int k = 0; k < 2 * KD; k++) {
      float2 y = make_float2(0.f, 0.f);
      if (r < hp.n && k * 8 < dim) {
        if (a.q_pairs)
          y = *reinterpret_cast<const float2*>(q + k * 8);
        else
          y = make_float2(q[k * 8], q[k * 8 + 1]);
      }
      x[k >> 1][(k & 1) * 2] = y.x;
      x[k >> 1][(k & 1) * 2 + 1] = y.y;
    }
#pragma unroll
    for (int k = 0; k < KD; k++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[k][i] *= a.scale;
        top = fmaxf(top, fabsf(x[k][i]));
      }
    float up = 1.f;
    unscale = 1.f;
    if constexpr (!H::THREE) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t ex = max(__float_as_uint(top) >> 23, 15u);  // (2^-112: a smaller q leaves the scores at 0)
      up = __uint_as_float((268 - ex) << 23);
      unscale = ex < 255 ? __uint_as_float((ex - 14) << 23) : NAN;  // NaN leads to attend_plain
    }
#pragma unroll
    for (int k = 0; k < KD; k++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t z = 0;
        parts(x[k][2 * i] * up, x[k][2 * i + 1] * up, qa[k][2 * i], qa[k][2 * i + 1], z);
        if constexpr (EXTRA) qb[k][i] = z;
      }
#pragma unroll
    for (int j = 0; j < 2 * KD; j++) acc[j][0] = acc[j][1] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  __device__ void tile(const AttendArgs&, char* st, uint32_t ok) {
    const int lane = threadIdx.x & 31, c = (lane & 3) * 2, sw = KD <= 2 ? (lane >> 1) & 3 : lane & 7;
    const uint32_t ks = smem_u32(st) + ((lane & 7) + (lane >> 4) * 8) * ROW, ku = (lane >> 3) & 1;
    const uint32_t vs = smem_u32(st) + SLABS * SLAB_BYTES + (lane & 15) * ROW, vu = lane >> 4;
    float s[NB][2];
#pragma unroll
    for (int h = 0; h < NB / 2; h++) {
      float d0[2][4] = {}, d1[2][4] = {};
#pragma unroll
      for (int k = 0; k < KD; k++) {
        uint32_t b[4];
        ldmatrix4(b, ks + h * 16 * ROW + k / 4 * SLAB_BYTES + (((k % 4 * 2 + ku) ^ sw) << 4));
        H::mma(d0[0], qa[k], b[0], b[1], d0[0]);
        H::mma(d0[1], qa[k], b[2], b[3], d0[1]);
        if constexpr (EXTRA) {
          const uint32_t low[4] = {qb[k][0], 0, qb[k][1], 0};
          H::mma(d1[0], low, b[0], b[1], d1[0]);
          H::mma(d1[1], low, b[2], b[3], d1[1]);
        }
      }
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float x = d0[n][i] + (H::THREE ? d0[n][2 + i] + (EXTRA ? d1[n][i] : 0.f) : d0[n][2 + i] * H::DOWN);
          if constexpr (SPLIT) x += __shfl_xor_sync(0xffffffffu, x, 16);
          s[2 * h + n][i] = H::THREE ? x : x * unscale;
        }
    }
    if (ok != 0xFFFFFFFFu >> (32 - KT)) {
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int i = 0; i < 2; i++)
          if (!((ok >> (n * 8 + c + i)) & 1)) s[n][i] = -INFINITY;
    }
    float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
    for (int n = 1; n < NB; n++) top = fmaxf(top, fmaxf(s[n][0], s[n][1]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (__any_sync(0xffffffffu, top > m + kLazy)) {
      const float to = fmaxf(m, H::THREE ? top : ceilf(top)), f = to == -INFINITY ? 1.f : exp2f(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int j = 0; j < 2 * KD; j++) acc[j][0] *= f, acc[j][1] *= f;
    }
    // fp16: the tile's own exponent, and the power of two that leads from there to m.  (2^14 is multiplied by:
    // added to the exponent it would round the small differences that the largest weights come from.)
    const float from = H::THREE ? (m == -INFINITY ? 0.f : m) : top == -INFINITY ? 0.f : ceilf(top);
    const float back = H::THREE ? 1.f : top == -INFINITY ? 0.f : exp2f(from - m) * 0x1p-14f;
    float sum = 0.f;
    uint32_t pa[NB / 2][4], pb[NB / 2][4] = {};
#pragma unroll
    for (int n = 0; n < NB; n++) {
      const float u = exp2f(s[n][0] - from) * (H::THREE ? 1.f : 0x1p14f);
      const float v = exp2f(s[n][1] - from) * (H::THREE ? 1.f : 0x1p14f);
      if constexpr (H::THREE)
        l += u + v;
      else
        sum += u + v;
      uint32_t(&x)[4] = pa[n / 2];
      parts(u, v, x[n % 2 * 2], x[n % 2 * 2 + 1], pb[n / 2][n % 2 * 2]);
    }
    if constexpr (!H::THREE) l += sum * back;
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KD; j++) {
      float d[2][4];
#pragma unroll
      for (int h = 0; h < NB / 2; h++) {
        uint32_t b[4];
        ldmatrix4_trans(b, vs + h * 16 * ROW + j / 4 * SLAB_BYTES + (((j % 4 * 2 + vu) ^ sw) << 4));
#pragma unroll
        for (int i = 0; i < 2; i++) {
          if (h == 0)
            H::mma(d[i], pa[h], b[2 * i], b[2 * i + 1], zero);
          else
            H::mma(d[i], pa[h], b[2 * i], b[2 * i + 1], d[i]);
          if constexpr (EXTRA) H::mma(d[i], pb[h], b[2 * i], b[2 * i + 1], d[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if constexpr (H::THREE) {
          acc[2 * j + i][0] += d[i][0] + d[i][2];
          acc[2 * j + i][1] += d[i][1] + d[i][3];
        } else {
          acc[2 * j + i][0] += (d[i][0] + d[i][2] * H::DOWN) * back;
          acc[2 * j + i][1] += (d[i][1] + d[i][3] * H::DOWN) * back;
        }
      }
    }
  }

  __device__ bool finish(const AttendArgs& a, float* rec) {
    const int r = row(), c = (threadIdx.x & 3) * 2, dim = a.kv.dim;
    const bool big = below_one(acc, m, l);
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if constexpr (SPLIT) {
#pragma unroll
      for (int j = 0; j < 2 * KD; j++)
#pragma unroll
        for (int i = 0; i < 2; i++) acc[j][i] += __shfl_xor_sync(0xffffffffu, acc[j][i], 16);
    }
    if (big && !all_finite(acc, l)) return false;
    if (r < a.part && !(SPLIT && (threadIdx.x & 16))) {
      float* x = rec + r * (dim + 2);
      if (c == 0) {
        x[0] = m;
        x[1] = l;
      }
#pragma unroll
      for (int j = 0; j < 2 * KD; j++)
        if (j * 8 < dim) {
          x[2 + j * 8 + c] = acc[j][0];
          x[3 + j * 8 + c] = acc[j][1];
        }
    }
    __syncwarp();
    return true;
  }
};

// ------------------------------------------------------- fp32 caches (and wide 16-bit heads)
//
// LPR lanes share a row, each with CPL units of 16 bytes of it, so a warp treats 32 / LPR positions at
// a time, R times per tile.  The R * GT partial
// scores of a lane are summed over the lanes of a row by halving: each step exchanges half of the
// values with a lane that keeps the other half, so 32 sums cost 31 shuffles and not 160, and each
// lane ends with the scores that it turns into weights (no weight is computed twice).
template <typename T, int LPR, int CPL, int GT>
struct PathFma {
  using Type = T;
  static constexpr int VE = 16 / (int)sizeof(T), KPW = 32 / LPR;
  static constexpr int KT = LPR <= 16 ? 16 : CPL == 1 ? 8 : 4, R = KT / KPW;
  static constexpr int WARPS = 8, MAX_DIM = LPR * CPL * VE;
  static constexpr bool RING = true;
  static constexpr int SWIZZLE = 0;
  static constexpr int SLAB = LPR * CPL * VE, SLABS = 1, PITCH = SLAB * (int)sizeof(T), SLAB_BYTES = KT * PITCH;
  static constexpr int TILE_BYTES = 2 * SLAB_BYTES;
  static constexpr int STAGE_BYTES = TILE_BYTES + (KT * GT * 4 + 127) / 128 * 128;
  static constexpr int STAGES = 2, BLOCKS = TILE_BYTES < 8192 && GT <= 4 ? 2 : 1;
  static constexpr int V = R * GT, NV = V > LPR ? V / LPR : 1;  // scores per lane
  static constexpr int SAME = LPR / GT;                         // lanes of a row with scores of one head
  static constexpr int COPIES = V < LPR ? LPR / V : 1;          // lanes of a row with the same score
  static_assert(GT <= LPR && R % 4 == 0, "layout");

  float q[GT][CPL * VE], acc[GT][CPL * VE], m, l;  // m, l: of this lane's head

  __device__ static int lane_in() { return (threadIdx.x & 31) % LPR; }
  __device__ static int group() { return (threadIdx.x & 31) / LPR; }
  __device__ static int first() { return V >= LPR ? lane_in() * NV : lane_in() / COPIES; }  // score index g * R + r

  __device__ void begin(const AttendArgs& a, int b, int hc) {
    const HeadPart hp = head_part(a, hc);
    const int dim = a.kv.dim;
#pragma unroll
    for (int g = 0; g < GT; g++) {
      const bool head = g < hp.n;
      const float* x = a.q + (size_t)b * a.qs + (size_t)(hp.head + (head ? g : 0)) * dim;
#pragma unroll
      for (int i = 0; i < CPL * VE; i++) {
        const int d = (lane_in() + (i / VE) * LPR) * VE + i % VE;
        q[g][i] = head && d < dim ? x[d] * a.scale : 0.f;
        acc[g][i] = 0.f;
      }
    }
    m = -INFINITY;
    l = 0.f;
  }

  static __device__ __forceinline__ void load(const char* at, float (&x)[CPL * VE]) {
#pragma unroll
    for (int c = 0; c < CPL; c++) {
      const uint4 u = *reinterpret_cast<const uint4*>(at + c * LPR * 16);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (VE == 4) {
          x[c * VE + i] = __uint_as_float(w[i]);
        } else {
          const float2 f = Half2<T>::unpack(w[i]);
          x[c * VE + 2 * i] = f.x;
          x[c * VE + 2 * i + 1] = f.y;
        }
      }
    }
  }

  template <int N, int O>
  static __device__ __forceinline__ void halve(float* v) {
    if constexpr (O > 0) {
      if constexpr (N > 1) {
        const bool up = (threadIdx.x & O) != 0;
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
          const float send = up ? v[i] : v[i + N / 2], keep = up ? v[i + N / 2] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, O);
        }
        halve<N / 2, O / 2>(v);
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], O);
        halve<1, O / 2>(v);
      }
    }
  }

  __device__ void tile(const AttendArgs&, char* st, uint32_t ok) {
    const char* rows = st + group() * PITCH + lane_in() * 16;
    float s[V];
#pragma unroll
    for (int r = 0; r < R; r++) {
      float k[CPL * VE];
      load(rows + r * KPW * PITCH, k);
#pragma unroll
      for (int g = 0; g < GT; g++) {
        float x = q[g][0] * k[0];
#pragma unroll
        for (int i = 1; i < CPL * VE; i++) x += q[g][i] * k[i];
        s[g * R + r] = x;
      }
    }
    halve<V, LPR / 2>(s);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int r = (first() + i) % R;
      if (!((ok >> (r * KPW + group())) & 1)) s[i] = -INFINITY;
      top = fmaxf(top, s[i]);
    }
#pragma unroll
    for (int o = 1; o < SAME; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (__any_sync(0xffffffffu, top > m + kLazy)) {
      const float to = fmaxf(m, top), f = to == -INFINITY ? 1.f : exp2f(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int g = 0; g < GT; g++) {
        const float fg = __shfl_sync(0xffffffffu, f, g * SAME);
#pragma unroll
        for (int i = 0; i < CPL * VE; i++) acc[g][i] *= fg;
      }
    }
    float* ps = reinterpret_cast<float*>(st + TILE_BYTES) + group() * V;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const float p = exp2_of(s[i], m);
      l += p;
      ps[first() + i] = p;
    }
    __syncwarp();
#pragma unroll
    for (int r4 = 0; r4 < R; r4 += 4) {
      float p[GT][4];
#pragma unroll
      for (int g = 0; g < GT; g++) *reinterpret_cast<float4*>(p[g]) = *reinterpret_cast<const float4*>(ps + g * R + r4);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float v[CPL * VE];
        load(rows + (KT + (r4 + r) * KPW) * PITCH, v);
#pragma unroll
        for (int g = 0; g < GT; g++)
#pragma unroll
          for (int i = 0; i < CPL * VE; i++) acc[g][i] += p[g][r] * v[i];
      }
    }
  }

  // (Not finite where the formula is: a weight of 0 times an infinite value, weights of up to 2^kLazy times values
  // near the largest.)
  __device__ bool finish(const AttendArgs& a, float* rec) {
    const int dim = a.kv.dim;
    const bool big = below_one(acc, m, l);
#pragma unroll
    for (int o = 1; o < SAME; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
      for (int g = 0; g < GT; g++)
#pragma unroll
        for (int i = 0; i < CPL * VE; i++) acc[g][i] += __shfl_xor_sync(0xffffffffu, acc[g][i], o);
    }
    if (big && !all_finite(acc, l)) return false;
    if (group() == 0) {
#pragma unroll
      for (int g = 0; g < GT; g++) {
        if (g >= a.part) continue;
        float* x = rec + g * (dim + 2);
        if (lane_in() == g * SAME) {
          x[0] = m;
          x[1] = l * (1.f / COPIES);
        }
#pragma unroll
        for (int i = 0; i < CPL * VE; i++) {
          const int d = (lane_in() + (i / VE) * LPR) * VE + i % VE;
          if (d < dim) x[2 + d] = acc[g][i];
        }
      }
    }
    __syncwarp();
    return true;
  }
};

// ------------------------------------------------------------------------------ the kernel
// The records of a warp: [0] a part that goes on from the stretch before, [1] one that begins in this stretch.
struct Records {
  float* rec;        // [2][rf]
  int rf;
  long long* id;     // where on the line the sequence part begins, -1: none
  int *b, *hc, *tiles;
};

// Positions of the tiles [t0, t1] of a sequence.
template <int KT>
__device__ __forceinline__ uint2 positions(const AttendArgs& a, const Seq& s, uint32_t t0, uint32_t t1) {
  uint32_t j0, j1, skip;
  tile_span<KT>(a, t0, &j0, &skip);
  tile_span<KT>(a, t1, &skip, &j1);
  return make_uint2(max(s.first, j0), min(s.n, j1));
}

// At the last tile of a sequence part that this warp sees: its record is the result, or goes to the joins.
template <int KT>
__device__ __forceinline__ void end_part(const AttendArgs& a, const Walk<KT>& at, bool starts, bool ends, const Records& r) {
  const int lane = threadIdx.x & 31, which = starts ? 1 : 0, dim = a.kv.dim;
  if (starts && ends) {
    const HeadPart hp = head_part(a, at.hc);
    for (int g = 0; g < hp.n; g++) {
      const float* x = r.rec + which * r.rf + g * (dim + 2);
      for (int d = lane; d < dim; d += 32) store_out(a, at.b, hp.head + g, d, x[2 + d], x[1]);
      if (lane == 0) store_lse(a, at.b, hp.head + g, x[0], x[1]);
    }
    __syncwarp();
  } else if (lane == 0) {
    r.id[which] = (long long)at.pos - (long long)(at.t - at.s.t0) - kPartCost;
    r.b[which] = at.b;
    r.hc[which] = at.hc;
    r.tiles[which] = at.s.t1 - at.s.t0;
  }
}

// The stretch [at, whi) by attend_plain: any layout, and once more where a path met something that is not
// finite or a copy that did not arrive in time.  A function of its own, behind the loop over tiles: a call inside that loop made it spill, which cost
// 16-bit heads of 16 and 32 and eight bf16 heads of 128 per key head half of their rate.
template <typename P>
__device__ __noinline__ void attend_stretch(const AttendArgs& a, Walk<P::KT> at, unsigned long long whi, Records r) {
  const int hcs = a.kv.kv_heads * a.chunks;
  while (true) {
    const uint32_t from = at.t, n = (uint32_t)min(whi - at.pos, (unsigned long long)(at.s.t1 - at.t));
    at.t += n - 1;
    at.pos += n - 1;
    const bool starts = from == at.s.t0, ends = at.t + 1 == at.s.t1;
    const uint2 j = positions<P::KT>(a, at.s, from, at.t);
    float* rec = r.rec + (starts ? r.rf : 0);
    if (P::MAX_DIM <= 64 || a.kv.dim <= 64)
      attend_plain<typename P::Type, 2, 4>(a, at.b, at.hc, j.x, j.y, rec);
    else
      attend_plain<typename P::Type, 8, 1>(a, at.b, at.hc, j.x, j.y, rec);
    end_part(a, at, starts, ends, r);
    if (at.pos + 1 + (ends ? kPartCost : 0) >= whi) return;
    at.next(a, hcs);
  }
}

template <typename P>
constexpr size_t ring_bytes() {
  return (size_t)P::WARPS * P::STAGES * (P::STAGE_BYTES + 16);  // stages, then barriers and row bits of each
}

template <typename P>
__global__ void __launch_bounds__(P::WARPS * 32, P::BLOCKS)
    k_paged_attend(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v) {
  constexpr int KT = P::KT, WARPS = P::WARPS, THREADS = WARPS * 32;
  static_assert(2 * WARPS <= 32, "a lane per record");
  extern __shared__ char smem_raw[];
  char* smem = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;  // the swizzle's period
  __shared__ unsigned long long pre[kPrefix];
  __shared__ unsigned long long warp_tot[WARPS];
  __shared__ uint32_t warp_long[WARPS], warp_live[WARPS];
  __shared__ long long seg_id[WARPS * 2];  // where on the line the sequence part of each record begins, -1: none
  __shared__ int seg_b[WARPS * 2], seg_hc[WARPS * 2], seg_tiles[WARPS * 2];
  __shared__ int open_first[2], open_parts[2], open_rec[2];  // parts that other blocks share: first block, blocks, record
  __shared__ unsigned s_old[2];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, dim = a.kv.dim;
  const int hcs = a.kv.kv_heads * a.chunks;
  const int rf = rec_floats(a.part, dim);
  float* recs = reinterpret_cast<float*>(smem + ring_bytes<P>());
  char* ring = smem + w * P::STAGES * P::STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WARPS * P::STAGES * P::STAGE_BYTES) + w * P::STAGES * 2;  // barrier, bits
  if constexpr (P::RING) {
    if (tid == 0) {
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
    }
    if (lane < P::STAGES) mbar_init(&bars[lane * 2], 1);
    mbar_fence_init();
    fence_async();
  }
  if (tid < WARPS * 2) seg_id[tid] = -1;
  if (tid < 2) open_first[tid] = -1;
  pdl_wait();
  pdl_trigger();

  // Places before every `step`-th sequence, the longest part, and how many parts there are.
  const int step = (a.kv.batch + kPrefix - 1) / kPrefix, n_pre = step == 1 ? a.kv.batch : (a.kv.batch + step - 1) / step;
  unsigned long long total = 0;
  uint32_t longest = 0, live_seqs = 0;
  for (int e0 = 0; e0 < n_pre; e0 += THREADS) {
    const int e = e0 + tid;
    unsigned long long sum = 0;
    uint32_t most = 0, live = 0;
    if (e < n_pre)
      for (int b = e * step; b < min(a.kv.batch, (e + 1) * step); b++) {
        const Seq s = seq_of<KT>(a, b);
        if (s.n == 0 && a.kv.lens[b] != 0 && blockIdx.x == 0) atomicExch(&a.flags[FLAG_RANGE], RANGE_PAGE);
        sum += s.n ? s.t1 - s.t0 + kPartCost : 0;
        most = max(most, s.t1 - s.t0);
        live += s.n != 0;
      }
    sum *= hcs;
    unsigned long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 31) {
      warp_tot[w] = inc;
      warp_long[w] = most;
      warp_live[w] = live;
    }
    __syncthreads();
    unsigned long long before = total + inc - sum;
#pragma unroll
    for (int i = 0; i < WARPS; i++) {
      const unsigned long long x = warp_tot[i];
      if (i < w) before += x;
      total += x;
      longest = max(longest, warp_long[i]);
      live_seqs += warp_live[i];
    }
    if (e < n_pre) pre[e] = before;
    __syncthreads();
  }

  // Idle sequences: zeros.
  if (live_seqs < (uint32_t)a.kv.batch)
    for (int b = blockIdx.x; b < a.kv.batch; b += gridDim.x) {
      if (seq_of<KT>(a, b).n) continue;
      for (int e = tid; e < a.heads * dim; e += THREADS) a.out[(size_t)b * a.os + e] = 0.f;
      if (a.lse)
        for (int e = tid; e < a.heads; e += THREADS) a.lse[(size_t)b * a.heads + e] = -INFINITY;
    }
  if (total == 0) return;

  // The first tile at place u of the line or behind it, and where its sequence part begins.
  auto locate = [&](unsigned long long u, Walk<KT>& at) -> unsigned long long {
    int l = 0;
    for (int n = n_pre; n > 1;) {  // the last entry <= u is among l .. l + n - 1: a 32nd of them per step
      const int piece = (n + 31) / 32, x = l + lane * piece;
      const int to = (31 - __clz(__ballot_sync(0xffffffffu, x < l + n && pre[x] <= u) | 1)) * piece;
      l += to;
      n = min(piece, n - to);
    }
    unsigned long long x = pre[l];
    auto places = [&]() { return at.s.n ? (unsigned long long)(at.s.t1 - at.s.t0 + kPartCost) * hcs : 0; };
    at.b = l * step;
    at.s = seq_of<KT>(a, at.b);
    while (x + places() <= u && at.b + 1 < a.kv.batch) {
      x += places();
      at.s = seq_of<KT>(a, ++at.b);
    }
    const uint32_t part = at.s.t1 - at.s.t0 + kPartCost;
    at.hc = (int)div64(u - x, part);  // (a long sequence times its key heads passes 32 bits)
    const uint32_t off = (uint32_t)(u - x - (unsigned long long)at.hc * part), tile = off > kPartCost ? off - kPartCost : 0;
    at.t = at.s.t0 + tile;
    at.pos = u - off + kPartCost + tile;
    return u - off;
  };

  // This block's stretch of the line, and this warp's.  Where every part of a sequence is short, blocks
  // take whole parts: the join between blocks costs more than the evenness gives.
  const bool whole = longest <= WARPS * a.whole_tiles;
  const unsigned long long want = whole ? (unsigned long long)live_seqs * hcs : div64(total, WARPS * a.min_tiles) + 1;
  const unsigned blocks = want < gridDim.x ? (unsigned)want : gridDim.x;
  const unsigned long long share = div64(total + blocks - 1, blocks);  // places per block
  unsigned long long lo = share * blockIdx.x, hi = min(lo + share, total);
  if (lo >= total) return;
  if (whole) {  // the parts that begin in the stretch
    Walk<KT> x;
    unsigned long long s0 = locate(lo, x);
    if (s0 != lo) lo = s0 + (x.s.t1 - x.s.t0) + kPartCost;
    s0 = locate(hi - 1, x);
    hi = max(hi, s0 + (x.s.t1 - x.s.t0) + kPartCost);
    if (lo >= hi) return;
    lo += kPartCost;  // where its first tile is
  }
  const uint32_t each = ((uint32_t)(hi - lo) + WARPS - 1) / WARPS;
  const unsigned long long wlo = min(lo + w * each, hi), whi = min(wlo + each, hi);

  Walk<KT> at;  // where the softmax is
  at.pos = whi;
  if (wlo < whi) locate(wlo, at);
  if (at.pos < whi) {
    const Records mine = {recs + w * 2 * rf, rf, seg_id + w * 2, seg_b + w * 2, seg_hc + w * 2, seg_tiles + w * 2};
    if constexpr (P::RING) {
      P path;
      bool again = false, late = false;  // late: a wait ran out, which is reported
      Walk<KT> ahead = at;  // where the copies are
      uint32_t stage_in = 0, stage_out = 0, parity = 0;
      // Lane i looks up the page of the i-th box of the next tile to issue, a tile early.
      const int boxes = a.page_tiles ? 1 : KT / a.box_rows;
      uint32_t id = 0, slot = 0, span0 = 0, span1 = 0;
      bool live = false;
      auto look = [&]() {
        tile_span<KT>(a, ahead.t, &span0, &span1);
        const uint32_t j = span0 + lane * a.box_rows;
        live = lane < boxes && j < ahead.s.n && j + a.box_rows > ahead.s.first;
        const uint32_t pg = live ? page_of(a, j) : 0;
        slot = j - pg * a.kv.page_size;
        id = live ? a.kv.table[(size_t)ahead.b * a.kv.max_pages + pg] : 0;
      };
      look();
      auto issue = [&]() {
        if (ahead.pos >= whi) return;
        const bool bad = live && id >= a.kv.n_pages;
        if (bad) atomicExch(&a.flags[FLAG_RANGE], RANGE_PAGE);
        // rows that are attended to: within the sequence, the window and (one box only) the page
        const uint32_t lo = ahead.s.first > span0 ? ahead.s.first - span0 : 0, hi = min(ahead.s.n, span1) - span0;
        uint32_t ok = ((2u << (hi - 1)) - 1) & ~((1u << lo) - 1);
        uint32_t lost = __ballot_sync(0xffffffffu, bad);
        while (lost) {
          const int x = __ffs(lost) - 1;
          lost &= lost - 1;
          ok &= ~((0xFFFFFFFFu >> (32 - a.box_rows)) << (x * a.box_rows));
        }
        char* st = ring + stage_in * P::STAGE_BYTES;
        uint64_t* bar = &bars[stage_in * 2];
        if (lane == 0) {
          bar[1] = ok;
          mbar_arrive_expect_tx(bar, 2 * P::SLABS * P::SLAB_BYTES);
        }
        __syncwarp();
        if (lane < boxes) {
          // a box without a page lies outside the tensor: zeros
          const int page = live && !bad ? (int)id : (int)a.kv.n_pages, hk = head_part(a, ahead.hc).kv;
          const uint32_t dst = smem_u32(st) + lane * a.box_rows * (P::SLAB_BYTES / KT);
#pragma unroll
          for (int c = 0; c < P::SLABS; c++) {
            tma_load_4d(dst + c * P::SLAB_BYTES, &tm_k, c * P::SLAB, (int)slot, hk, page, bar);
            tma_load_4d(dst + (P::SLABS + c) * P::SLAB_BYTES, &tm_v, c * P::SLAB, (int)slot, hk, page, bar);
          }
        }
        stage_in = stage_in + 1 == P::STAGES ? 0 : stage_in + 1;
        ahead.next(a, hcs);
        if (ahead.pos < whi) look();
      };
      for (int i = 0; i < P::STAGES - 1; i++) issue();
      uint32_t part_t = at.t;  // where this warp's share of the current sequence part begins
      path.begin(a, at.b, at.hc);
      for (bool more = true; more;) {
        issue();
        char* st = ring + stage_out * P::STAGE_BYTES;
        if (!__all_sync(0xffffffffu, mbar_wait(&bars[stage_out * 2], parity, a.flags, kWaitSite))) {
          again = late = true;
          break;
        }
        const uint32_t ok = (uint32_t)bars[stage_out * 2 + 1];
        if (ok != 0xFFFFFFFFu >> (32 - KT)) {
          // what the cache holds behind a sequence's end may be NaN, and 0 * NaN is not 0
          constexpr int ROW = P::SLAB_BYTES / KT;
          for (int e = lane * 16; e < P::SLABS * P::SLAB_BYTES; e += 512)
            if (!((ok >> (e % P::SLAB_BYTES / ROW)) & 1))
              *reinterpret_cast<uint4*>(st + P::SLABS * P::SLAB_BYTES + e) = make_uint4(0, 0, 0, 0);
          fence_async();
          __syncwarp();
        }
        path.tile(a, st, ok);
        __syncwarp();
        if (++stage_out == P::STAGES) {
          stage_out = 0;
          parity ^= 1;
        }
        const bool ends = at.t + 1 == at.s.t1;
        more = at.pos + 1 + (ends ? kPartCost : 0) < whi;
        if (ends || !more) {
          const bool starts = part_t == at.s.t0;
          if (!path.finish(a, mine.rec + (starts ? rf : 0))) {
            again = true;
            break;
          }
          end_part(a, at, starts, ends, mine);
          if (more) {
            at.next(a, hcs);
            part_t = at.t;
            path.begin(a, at.b, at.hc);
          }
        } else {
          at.t++;
          at.pos++;
        }
      }
      if (again) {
        // the copies under way land first, within another wait each: the joins use the ring's memory
        for (; late || stage_out != stage_in; late = false) {
          (void)mbar_wait(&bars[stage_out * 2], parity, a.flags, kWaitSite);
          if (++stage_out == P::STAGES) {
            stage_out = 0;
            parity ^= 1;
          }
        }
        locate(wlo, at);
        attend_stretch<P>(a, at, whi, mine);
      }
    } else {
      attend_stretch<P>(a, at, whi, mine);
    }
  }
  __syncthreads();

  // Join the warps' records, in the order of positions.  Records r = 2 w + which of one sequence part
  // follow one another; lane r holds record r's id, so every warp knows the runs.  A warp joins one
  // head of one run at a time.  A part that lies in this block whole is done; the block's first may have
  // begun before it (slot 0), its last may go on behind it (slot 1).
  const long long my_id = lane < 2 * WARPS ? seg_id[lane] : -1;
  const uint32_t used = __ballot_sync(0xffffffffu, my_id >= 0);
  const uint32_t below = used & ((1u << lane) - 1);
  const long long prev = __shfl_sync(0xffffffffu, my_id, below ? 31 - __clz(below) : 0);
  uint32_t left = __ballot_sync(0xffffffffu, my_id >= 0 && (!below || prev != my_id));
  bool any_open = false;
  for (int item = 0; left;) {
    const int r0 = __ffs(left) - 1;
    left &= left - 1;
    const uint32_t mine = used & (left ? (1u << (__ffs(left) - 1)) - 1 : 0xffffffffu) & ~((1u << r0) - 1);
    const HeadPart hp = head_part(a, seg_hc[r0]);
    const unsigned long long u0 = seg_id[r0] + kPartCost, u1 = u0 + seg_tiles[r0];  // its tiles
    const bool before = u0 < lo, open = before || u1 > hi;
    any_open |= open;
    if (open && tid == 0) {
      // blocks that hold tiles u0 and u1 - 1
      const int slot = before ? 0 : 1, c0 = (int)div64(u0, share);
      open_first[slot] = c0;
      open_parts[slot] = (int)div64(u1 - 1, share) - c0 + 1;
      open_rec[slot] = r0;
    }
    for (int g = 0; g < hp.n; g++, item++) {
      if (item % WARPS != w) continue;
      const float* rec = recs + g * (dim + 2);
      float m = -INFINITY, l = 0.f, o[8] = {};
      if ((mine >> lane) & 1) {
        m = rec[lane * rf];
        l = rec[lane * rf + 1];
      }
      const float top = warp_max(m), f = weight_of(m, l, top), sum = warp_sum(f * l);
      for (uint32_t x = mine; x; x &= x - 1) {
        const int r = __ffs(x) - 1;
        const float fx = __shfl_sync(0xffffffffu, f, r), *p = rec + r * rf + 2 + lane;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (lane + 32 * k < dim) o[k] += fx * p[32 * k];
      }
      if (open) {
        float* part = a.partial + (size_t)(blockIdx.x * 2 + (before ? 0 : 1)) * rf + g * (dim + 2);
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (lane + 32 * k < dim) __stcg(part + 2 + lane + 32 * k, o[k]);
        if (lane == 0) {
          __stcg(part, top);
          __stcg(part + 1, sum);
        }
      } else {
        store_head(a, seg_b[r0], hp.head + g, lane, o, top, sum);
      }
    }
  }
  if (!any_open) return;
  __syncthreads();
  // The block's results, which the barrier orders before, then the count, then anyone's reads of the
  // other blocks' results.
  if (tid < 2 && open_first[tid] >= 0) s_old[tid] = add_acq_rel(&a.counters[open_first[tid]]);
  __syncthreads();
  // Where this is the last block to arrive, every partial result is there: block c0's slot 1, then slot 0
  // of the next ones.  They are brought to shared memory (the ring's, and the records' behind it), one trip
  // to L2 for all of them where they fit; then a warp joins a head.  Two parts are joined at a time where
  // there are warps for both.
  float* stage = reinterpret_cast<float*>(smem);
  const int rf4 = rf / 4, most = 2 * WARPS + (int)(ring_bytes<P>() / 4) / rf;
  uint32_t todo = 0;
  for (int i = 0; i < 2; i++)
    if (open_first[i] >= 0 && s_old[i] + 1 == (unsigned)open_parts[i]) todo |= 1u << i;
  while (todo) {
    const bool both = todo == 3 && 2 * a.part <= WARPS && open_parts[0] + open_parts[1] <= most;
    const int i0 = both ? 0 : __ffs(todo) - 1, first = open_parts[i0], parts = both ? first + open_parts[1] : first;
    const int mine = both && w >= WARPS / 2 ? 1 : i0, g = both ? w % (WARPS / 2) : w;
    const HeadPart hp = head_part(a, seg_hc[open_rec[mine]]);
    todo = both ? 0 : todo & (todo - 1);
    const int from = open_first[i0], from1 = open_first[1];
    const uint32_t mul = 0xFFFFFFFFu / rf4 + 1;  // e / rf4 = umulhi(e, mul), e < 2^16, rf4 > 1
    float o[8] = {}, top = -INFINITY, sum = 0.f;
    for (int x0 = 0; x0 < parts; x0 += most) {
      const int n = min(most, parts - x0);
      __syncthreads();
      // eight loads under way per thread: one after another they took 35 us for 74 parts of 8 heads of 128
      for (int e0 = tid; e0 < n * rf4; e0 += 8 * THREADS) {
        float4 v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const int e = min(e0 + u * THREADS, n * rf4 - 1), r = (int)__umulhi((uint32_t)e, mul), x = x0 + r;
          const int y = x < first ? x : x - first, at = ((x < first ? from : from1) + y) * 2 + (y == 0);
          v[u] = __ldcg(reinterpret_cast<const float4*>(a.partial + (size_t)at * rf) + e - r * rf4);
        }
#pragma unroll
        for (int u = 0; u < 8; u++)
          if (e0 + u * THREADS < n * rf4) reinterpret_cast<float4*>(stage)[e0 + u * THREADS] = v[u];
      }
      __syncthreads();
      if (g < hp.n) {
        const float* rec = stage + (mine != i0 ? first * rf : 0) + g * (dim + 2);
        const int count = both ? open_parts[mine] : n;
        for (int y0 = 0; y0 < count; y0 += 32) {
          const int ny = min(32, count - y0);
          float m = -INFINITY, l = 0.f;
          if (lane < ny) {
            m = rec[(y0 + lane) * rf];
            l = rec[(y0 + lane) * rf + 1];
          }
          const float to = fmaxf(top, warp_max(m)), back = weight_of(top, sum, to), f = weight_of(m, l, to);
          sum = sum * back + warp_sum(f * l);
          top = to;
#pragma unroll
          for (int k = 0; k < 8; k++) o[k] *= back;
#pragma unroll 4  // (left to the compiler: once 38 us, once 43, for 148 parts of 8 heads of 32)
          for (int y = 0; y < ny; y++) {
            const float fx = __shfl_sync(0xffffffffu, f, y), *p = rec + (y0 + y) * rf + 2 + lane;
#pragma unroll
            for (int k = 0; k < 8; k++)
              if (lane + 32 * k < dim) o[k] += fx * p[32 * k];
          }
        }
      }
    }
    if (g < hp.n) store_head(a, seg_b[open_rec[mine]], hp.head + g, lane, o, top, sum);
    if (tid == 0) {
      a.counters[open_first[i0]] = 0;
      if (both) a.counters[open_first[1]] = 0;
    }
  }
}

// Tensor map of a paged cache: [page][head][slot][dim], boxes of `rows` slots x `cols` elements.
int cache_map(CUtensorMap* map, const void* base, int dtype, const PagedLayout& kv, int cols, int rows, int swizzle) {
  const TensorMapEncode enc = tensor_map_encode();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled entry point unavailable");
    return ERR_CUDA;
  }
  const size_t es = cache_type_size(dtype);
  cuuint64_t dims[4] = {(cuuint64_t)kv.dim, kv.page_size, (cuuint64_t)kv.kv_heads, kv.n_pages};
  cuuint64_t strides[3] = {kv.slot_stride * es, kv.head_stride * es, kv.page_stride * es};
  cuuint32_t box[4] = {(cuuint32_t)cols, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = enc(map,
                         dtype == TURT_CACHE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                         : dtype == TURT_CACHE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                         4, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                         : swizzle == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                         : CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (code " + std::to_string((int)r) + ")");
    return ERR_CUDA;
  }
  return OK;
}

template <typename P>
int attend_launch(turt_ctx* ctx, AttendArgs a, int part) {
  static std::atomic<uint64_t> done{0};
  a.part = part;
  a.chunks = (a.group + part - 1) / part;
  // At least 32 positions per warp (1 x 1000 positions, 6 fp32 heads of 64: 10.3 us, with 64 at least 13.4);
  // whole parts in a block where the longest has up to 64 per warp (1 x 200: 7.4 us, cut up 11.1; but 16 x
  // 1 .. 1000, 32 / 8 bf16 heads of 128: 17.3 us cut up, 19.9 whole).
  a.min_tiles = std::max(1, 32 / P::KT);
  a.whole_tiles = std::min(4, 64 / P::KT);
  a.box_rows = P::KT;
  a.page_tiles = 0;
  CUtensorMap tm_k{}, tm_v{};
  if constexpr (P::RING) {
    // a tile is one box or several (of 8 rows at least, the swizzle's period), or, for page sizes that
    // these do not divide, what a page has of it
    const int ps = (int)a.kv.page_size;
    while (a.box_rows > (P::SWIZZLE ? 8 : 4) && ps % a.box_rows) a.box_rows /= 2;
    if (ps % a.box_rows) {
      a.box_rows = P::KT;
      a.page_tiles = (ps + P::KT - 1) / P::KT;
    }
    RC(cache_map(&tm_k, a.kc, a.dtype, a.kv, P::SLAB, a.box_rows, P::SWIZZLE));
    RC(cache_map(&tm_v, a.vc, a.dtype, a.kv, P::SLAB, a.box_rows, P::SWIZZLE));
  }
  int sms = 0;
  RC(sm_count(ctx->device, &sms));
  const size_t rec = (size_t)P::WARPS * 2 * rec_floats(part, a.kv.dim) * 4, smem = ring_bytes<P>() + rec + 1024;
  RC(smem_attr_per_device(done, k_paged_attend<P>, 218 * 1024));
  TURT_REQUIRE(smem <= 218 * 1024, "paged_attention: shared memory");
  const int per_sm = smem <= 104 * 1024 ? P::BLOCKS : 1;
  const int grid = std::min(kMaxBlocks, sms * per_sm);
  TURT_CHECK_CUDA(launch_pdl(k_paged_attend<P>, dim3(grid), dim3(P::WARPS * 32), smem, ctx->stream, a, tm_k, tm_v));
  TURT_LAUNCH_CHECK();
  return OK;
}

// Whether bulk tensor copies can read the cache: rows of whole 16-byte units on 16-byte boundaries, and
// strides of which each divides the next larger one.
template <typename T>
bool in_boxes(const AttendArgs& a) {
  const size_t n = 16 / sizeof(T);
  const PagedLayout& kv = a.kv;
  size_t s[3] = {kv.slot_stride, kv.head_stride, kv.page_stride};
  std::sort(s, s + 3);
  return aligned16(a.kc) && aligned16(a.vc) && kv.dim % n == 0 && s[0] > 0 && s[0] % n == 0 && s[1] % s[0] == 0 &&
         s[2] % s[1] == 0 && s[2] * sizeof(T) < ((size_t)1 << 40);
}

template <typename T, int LPR, int CPL, int MOST>
int attend_fma(turt_ctx* ctx, const AttendArgs& a) {
  if (a.group == 1) return attend_launch<PathFma<T, LPR, CPL, 1>>(ctx, a, 1);
  if (a.group == 2) return attend_launch<PathFma<T, LPR, CPL, 2>>(ctx, a, 2);
  if (a.group <= 4 || MOST == 4) return attend_launch<PathFma<T, LPR, CPL, 4>>(ctx, a, std::min(a.group, 4));
  if constexpr (MOST == 8) return attend_launch<PathFma<T, LPR, CPL, 8>>(ctx, a, std::min(a.group, 8));
  return ERR_UNSUPPORTED;
}

template <typename T, int KD>
int attend_mma(turt_ctx* ctx, const AttendArgs& a) {
  const int part = std::min(a.group, kGroup);
  if constexpr (Half2<T>::THREE)
    if (part <= 4) return attend_launch<PathMma<T, KD, true>>(ctx, a, part);
  return attend_launch<PathMma<T, KD, false>>(ctx, a, part);
}

template <typename T>
int attend_typed(turt_ctx* ctx, const AttendArgs& a) {
  const int dim = a.kv.dim;
  if (!in_boxes<T>(a)) return attend_launch<PathPlain<T>>(ctx, a, std::min(a.group, kGroup));
  if constexpr (sizeof(T) == 4) {
    if (dim <= 32) return attend_fma<T, 8, 1, 8>(ctx, a);
    if (dim <= 64) return attend_fma<T, 16, 1, 8>(ctx, a);
    if (dim <= 128) return attend_fma<T, 32, 1, 8>(ctx, a);
    return attend_fma<T, 32, 2, 4>(ctx, a);
  } else {
    if (dim <= 32) return attend_mma<T, 2>(ctx, a);
    if (dim <= 64) return attend_mma<T, 4>(ctx, a);
    if (dim <= 80) return attend_mma<T, 5>(ctx, a);
    if (dim <= 96) return attend_mma<T, 6>(ctx, a);
    if (dim <= 128) return attend_mma<T, 8>(ctx, a);
    return attend_fma<T, 32, 1, 4>(ctx, a);
  }
}

constexpr size_t kCounterBytes = kMaxBlocks * 4;

}  // namespace
}  // namespace turt

using namespace turt;

extern "C" int turt_paged_attention_workspace(const turt_paged_kv* kv, int n_head, size_t* bytes) {
  PagedLayout p;
  RC(paged_layout(kv, &p));
  TURT_REQUIRE(bytes, "paged_attention_workspace: null bytes");
  TURT_REQUIRE(n_head > 0 && n_head % kv->n_kv_head == 0, "paged_attention: n_head must be a multiple of n_kv_head");
  const int part = std::min(kGroup, n_head / kv->n_kv_head);
  *bytes = kCounterBytes + (size_t)kMaxBlocks * 2 * rec_floats(part, kv->head_dim) * 4;
  return OK;
}

extern "C" int turt_paged_attention(turt_ctx* ctx, const turt_paged_kv* kv, const float* q, size_t q_stride, float* out,
                                    size_t out_stride, float* lse, int n_head, float scale, int window, void* workspace,
                                    size_t workspace_bytes) {
  AttendArgs a;
  size_t need = 0;
  RC(paged_layout(kv, &a.kv));
  RC(turt_paged_attention_workspace(kv, n_head, &need));
  const size_t wide = (size_t)n_head * kv->head_dim;
  TURT_REQUIRE(kv->batch == 0 || (q && out), "paged_attention: null pointer");
  TURT_REQUIRE(kv->batch <= 1 || (q_stride >= wide && out_stride >= wide),
               "paged_attention: row strides below the row width");
  TURT_REQUIRE(window >= 0, "paged_attention: negative window");
  TURT_REQUIRE(isfinite(scale), "paged_attention: scale must be finite");
  TURT_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)lse) % 4 == 0, "paged_attention: misaligned pointer");
  TURT_REQUIRE(workspace && workspace_bytes >= need && aligned16(workspace),
               "paged_attention: workspace missing, misaligned or smaller than turt_paged_attention_workspace says");
  TURT_REQUIRE(ctx, "null context");
  TURT_CHECK_CUDA(cudaSetDevice(ctx->device));
  if (kv->batch == 0) return OK;
  a.kc = kv->k, a.vc = kv->v;
  a.q = q, a.out = out, a.lse = lse;
  a.qs = q_stride, a.os = out_stride;
  a.heads = n_head, a.group = n_head / kv->n_kv_head, a.window = window;
  a.scale = (float)(scale * 1.4426950408889634);
  // division by the page size: mul = ceil(2^(31 + s) / d) with 2^s >= d is exact for positions < 2^31
  int s = 0;
  while ((1ll << s) < kv->page_size) s++;
  a.div_mul = (uint32_t)(((1ull << (31 + s)) + kv->page_size - 1) / kv->page_size);
  a.div_shift = 31 + s;
  a.counters = static_cast<uint32_t*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  a.flags = ctx->flags;
  a.dtype = kv->dtype;
  a.q_pairs = (uintptr_t)q % 8 == 0 && q_stride % 2 == 0;
  if (kv->dtype == TURT_CACHE_F32) return attend_typed<float>(ctx, a);
  if (kv->dtype == TURT_CACHE_F16) return attend_typed<__half>(ctx, a);
  return attend_typed<__nv_bfloat16>(ctx, a);
}
