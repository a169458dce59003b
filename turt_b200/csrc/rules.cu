// rules.cu -- per-request rules on the logits of the next token: penalties for repeated tokens,
// biases and grammar masks.
//
//   n = times that id v was generated in row r;  seen = v in the prompt or generated
//   x = logits;  seen: x = x > 0 ? x / rep : x * rep;  n > 0: x -= freq * n, x -= pres;
//   x += bias[v];  mask bit 0: x = -infinity
//
// One pass over the logits, bound by their memory traffic.  A block owns a slice of one row's
// vocabulary and asks for all of its logits and mask bits at once.  While they arrive it counts the
// row's ids that fall into the slice in shared memory (integer atomics: the counts do not depend on
// their order) and lists each touched id once; then a thread per touched id, and not the stream, works
// out the new logit, which takes the count's place; the stream only picks it up.  Every block of a row
// reads all of the row's ids, from L2, which is why slices are as long as filling the GPU allows.
#include "../../include/turt_cuda.h"
#include <algorithm>

#include "ctx.cuh"

namespace turt {
namespace {

// Count word: in the prompt, has a bias (k_logit_rules_stream), and times generated.
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kTimes = 0x3FFFFFFFu;
constexpr uint32_t kNoMask = 0xFFFFFFFFu;

struct RuleArgs {
  turt_logit_rules r;
  const float* in;
  float* out;
  size_t ld, out_ld;
  int vocab;
  int* flags;
};

struct RowRules {
  float rep, freq, pres;
};

__device__ __forceinline__ float penalise(const RowRules& w, float x, uint32_t c) {
  if (c & ~kBiased) x = x > 0.f ? x / w.rep : x * w.rep;
  const uint32_t n = c & kTimes;
  if (n) {
    x -= w.freq * (float)n;
    x -= w.pres;
  }
  return x;
}

// Slices are cut where a float4 of the row starts: `lead` elements lie between that boundary and the
// row's first, so position e of the slice is id s0 + e.  VEC: in and out share their boundaries.
template <int THREADS, int NV, bool VEC>
__global__ void __launch_bounds__(THREADS, 1536 / THREADS) k_logit_rules(const __grid_constant__ RuleArgs a) {
  constexpr int SLICE = THREADS * NV * 4;
  extern __shared__ __align__(16) uint32_t cnt[];  // [SLICE] counts, then new logits
  uint32_t* touched = cnt + SLICE;                 // a bit per id with a new logit
  uint16_t* list = reinterpret_cast<uint16_t*>(touched + SLICE / 32);
  __shared__ uint32_t n_list;
  const int r = blockIdx.y, V = a.vocab, tid = threadIdx.x;
  const float* in = a.in + (size_t)r * a.ld;
  float* out = a.out + (size_t)r * a.out_ld;
  const int lead = VEC ? (int)((reinterpret_cast<uintptr_t>(in) >> 2) & 3) : 0;
  const int s0 = blockIdx.x * SLICE - lead;
  if (s0 >= V) return;
  const bool listed = a.r.tokens != nullptr || a.r.bias_ids != nullptr;
  if (listed) {
#pragma unroll
    for (int k = 0; k < NV; k++) *reinterpret_cast<uint4*>(cnt + (k * THREADS + tid) * 4) = make_uint4(0, 0, 0, 0);
    for (int e = tid; e < SLICE / 32; e += THREADS) touched[e] = 0;
    if (tid == 0) n_list = 0;
  }
  pdl_wait();
  pdl_trigger();
  bool bad = false;
  const uint32_t* mask = nullptr;
  if (a.r.mask) {
    const uint32_t m = a.r.mask_row ? a.r.mask_row[r] : (uint32_t)r;
    if (m < (uint32_t)a.r.n_masks)
      mask = a.r.mask + (size_t)m * ((V + 31) / 32);
    else if (m != kNoMask)
      bad = true;
  }
  float4 x[NV];
  uint32_t open[NV];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int id = s0 + (k * THREADS + tid) * 4;
    if (VEC && id >= 0 && id + 4 <= V) {
      x[k] = *reinterpret_cast<const float4*>(in + id);
    } else {
      x[k].x = id >= 0 && id < V ? in[id] : 0.f;
      x[k].y = id + 1 >= 0 && id + 1 < V ? in[id + 1] : 0.f;
      x[k].z = id + 2 >= 0 && id + 2 < V ? in[id + 2] : 0.f;
      x[k].w = id + 3 >= 0 && id + 3 < V ? in[id + 3] : 0.f;
    }
    open[k] = 0xF;
    if (mask && id < V) {
      const int at = max(id, 0), word = at >> 5, words = (V + 31) >> 5;
      const uint32_t low = mask[word], high = (at & 31) > 28 && word + 1 < words ? mask[word + 1] : 0;
      open[k] = __funnelshift_r(low, high, at & 31) << (at - id);
    }
  }
  if (listed) {
    __syncthreads();
    if (a.r.tokens) {
      const uint32_t i0 = a.r.token_start[r], i1 = a.r.token_start[r + 1];
      const uint32_t g = a.r.generated_start ? a.r.generated_start[r] : 0xFFFFFFFFu;
      auto count = [&](uint32_t i, uint32_t id) {
        const uint32_t e = id - (uint32_t)s0;
        bad |= id >= (uint32_t)V;
        if (e < (uint32_t)SLICE && id < (uint32_t)V) {
          const uint32_t old = i >= g ? atomicAdd(&cnt[e], 1u) : atomicOr(&cnt[e], kSeen);
          if (old == 0) list[atomicAdd(&n_list, 1u)] = (uint16_t)e;
        }
      };
      // four ids at a time where they lie in one 16-byte unit
      const uint32_t skew = (uint32_t)(reinterpret_cast<uintptr_t>(a.r.tokens) >> 2) & 3;
      for (uint64_t q = ((uint64_t)i0 + skew) / 4 + tid; q * 4 < (uint64_t)i1 + skew; q += THREADS) {
        const int64_t i = (int64_t)(q * 4) - skew;
        if (i >= i0 && i + 4 <= i1) {
          const uint4 u = *reinterpret_cast<const uint4*>(a.r.tokens + i);
          count((uint32_t)i, u.x);
          count((uint32_t)i + 1, u.y);
          count((uint32_t)i + 2, u.z);
          count((uint32_t)i + 3, u.w);
        } else {
          for (int64_t x = max(i, (int64_t)i0); x < min(i + 4, (int64_t)i1); x++) count((uint32_t)x, a.r.tokens[x]);
        }
      }
    }
    uint32_t b0 = 0, b1 = 0;
    bool wild = false;  // bias ids that do not increase
    if (a.r.bias_ids) {
      b0 = a.r.bias_start[r];
      b1 = a.r.bias_start[r + 1];
      for (uint32_t i = b0 + tid; i < b1; i += THREADS) {
        const uint32_t id = a.r.bias_ids[i], e = id - (uint32_t)s0;
        bad |= id >= (uint32_t)V;
        wild |= i > b0 && a.r.bias_ids[i - 1] >= id;
        if (e < (uint32_t)SLICE && id < (uint32_t)V) atomicOr(&touched[e >> 5], 1u << (e & 31));
      }
    }
    RowRules w;
    w.rep = a.r.repetition ? a.r.repetition[r] : 1.f;
    w.freq = a.r.frequency ? a.r.frequency[r] : 0.f;
    w.pres = a.r.presence ? a.r.presence[r] : 0.f;
    if (__syncthreads_or(wild)) {
      // an id that comes twice would belong to two threads: the row takes none of its biases
      bad = true;
      b1 = b0;
      for (int e = tid; e < SLICE / 32; e += THREADS) touched[e] = 0;
      __syncthreads();
    }
    // ids with a bias (their bits are set already) belong to it, the others to the list
    for (uint32_t i = b0 + tid; i < b1; i += THREADS) {
      const uint32_t id = a.r.bias_ids[i], e = id - (uint32_t)s0;
      if (e < (uint32_t)SLICE && id < (uint32_t)V)
        cnt[e] = __float_as_uint(penalise(w, in[id], cnt[e]) + a.r.bias[i]);
    }
    for (uint32_t i = tid; i < n_list; i += THREADS) {
      const uint32_t e = list[i], bit = 1u << (e & 31);
      if (!(atomicOr(&touched[e >> 5], bit) & bit))
        cnt[e] = __float_as_uint(penalise(w, in[(int)e + s0], cnt[e]));
    }
    __syncthreads();
  }
  if (bad) atomicExch(&a.flags[FLAG_RANGE], RANGE_RULE);
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int e = (k * THREADS + tid) * 4, id = s0 + e;
    if (id >= V) break;
    if (listed) {
      const uint32_t t = touched[e >> 5] >> (e & 31);
      if (t & 0xF) {
        const float4 y = *reinterpret_cast<const float4*>(cnt + e);
        if (t & 1) x[k].x = y.x;
        if (t & 2) x[k].y = y.y;
        if (t & 4) x[k].z = y.z;
        if (t & 8) x[k].w = y.w;
      }
    }
    if (!(open[k] & 1)) x[k].x = -INFINITY;
    if (!(open[k] & 2)) x[k].y = -INFINITY;
    if (!(open[k] & 4)) x[k].z = -INFINITY;
    if (!(open[k] & 8)) x[k].w = -INFINITY;
    if (VEC && id >= 0 && id + 4 <= V) {
      *reinterpret_cast<float4*>(out + id) = x[k];
    } else {
      if (id >= 0) out[id] = x[k].x;
      if (id + 1 >= 0 && id + 1 < V) out[id + 1] = x[k].y;
      if (id + 2 >= 0 && id + 2 < V) out[id + 2] = x[k].z;
      if (id + 3 >= 0 && id + 3 < V) out[id + 3] = x[k].w;
    }
  }
}

template <int THREADS, int NV>
int rules_launch(cudaStream_t st, const RuleArgs& a, int rows, bool vec) {
  static std::atomic<uint64_t> done{0}, done_vec{0};
  constexpr int SLICE = THREADS * NV * 4, SMEM = SLICE * 4 + SLICE / 8 + SLICE * 2;
  const dim3 grid(ceil_div((long)a.vocab + 3, SLICE), rows);
  if (vec) {
    RC(smem_attr_per_device(done_vec, k_logit_rules<THREADS, NV, true>, SMEM));
    TURT_CHECK_CUDA(launch_pdl(k_logit_rules<THREADS, NV, true>, grid, dim3(THREADS), SMEM, st, a));
  } else {
    RC(smem_attr_per_device(done, k_logit_rules<THREADS, NV, false>, SMEM));
    TURT_CHECK_CUDA(launch_pdl(k_logit_rules<THREADS, NV, false>, grid, dim3(THREADS), SMEM, st, a));
  }
  TURT_LAUNCH_CHECK();
  return OK;
}

// The same rules for large batches, as a pipeline: one block per SM walks over slices of up to
// kMostIds ids; a producer warp brings the logits, the row's ids, its biases and its mask bits of the
// slices ahead into a ring of shared memory, sixteen warps work in place on the slice that has
// arrived and store it.  The blocks of k_logit_rules wait for their ids, then for the touched logits,
// with nothing else to do; here both lie in shared memory before they are wanted.  When a block comes to
// a row of several slices it sorts the row's ids by slice once, so that each slice sees only its own (80 ->
// 65 us for 256 rows x 128000 ids with 4000 known ids a row).  Measured there, with 300 biases and masks: 69 us,
// 3.9 TB/s, against 44 us without any rule: sort, count, apply and mask of a slice follow one another between
// barriers on the same warps, 4200 cycles per 8000 ids where the memory would need 3000.  Slices as long as
// shared memory allows: 5120 ids and a longer ring took 94 us.
constexpr int kMostIds = 8192, kRing = 3, kWorkers = 512;
constexpr int kTokenRoom = 4096, kBiasRoom = 512;  // per slice; what is beyond is read from L2
constexpr int kSorted = 64;                        // slices of a row up to which its ids are sorted
constexpr int kWaitSite = 41;                      // reported when a wait of the pipeline runs out

struct RuleSlice {
  int row, s0;                // id of the slice's first position (negative: before the row)
  uint32_t i0, i1, made;      // ids of the row; from `made` on generated
  uint32_t b0, b1;            // biases
  uint32_t word0;             // first mask word here
  int masked;
  RowRules w;
};

struct __align__(128) RuleStage {
  float x[kMostIds];
  uint32_t tokens[kTokenRoom + 8];
  uint32_t bias_ids[kBiasRoom + 8];
  float bias[kBiasRoom + 8];
  uint32_t mask[kMostIds / 32 + 8];
  RuleSlice s;
};

struct RuleShared {
  RuleStage ring[kRing];
  uint32_t cnt[kMostIds];  // all zero between slices
  uint16_t list[kMostIds];
  uint32_t sorted[kTokenRoom];  // ids by slice, bit 31: generated
  uint32_t bins[kSorted + 1];   // sizes, then where each slice's ids begin
  uint64_t full[kRing], empty[kRing];
  uint32_t n_list[2];  // by turns
};

// Words between a place and the 16-byte boundary before it.
__device__ __forceinline__ uint32_t skew_of(const void* p) { return (uint32_t)(reinterpret_cast<uintptr_t>(p) >> 2) & 3; }

// n words on their way to dst, which lies as far from a 16-byte boundary as src: whole 16-byte units by
// one bulk copy counted by bar, the words at the ends through the registers of one warp.  They are
// asked for (ask) well before they are stored (put), or the producer would wait for memory once per array.
struct Bring {
  uint32_t* dst;
  const uint32_t* src;
  uint32_t head, body, tail, word;
  __device__ __forceinline__ void ask(void* d, const void* s, uint32_t n, int lane) {
    dst = static_cast<uint32_t*>(d);
    src = static_cast<const uint32_t*>(s);
    head = min((4 - skew_of(s)) & 3, n);
    body = (n - head) & ~3u;
    tail = n - head - body;
    const uint32_t at = lane < 4 ? lane : head + body + lane - 4;
    if (lane < head || (lane >= 4 && lane - 4 < tail)) word = src[at];
  }
  __device__ __forceinline__ void put(uint64_t* bar, int lane) const {
    if (body && lane == 0) {
      asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(body * 4) : "memory");
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       smem_u32(dst + head)),
                   "l"(src + head), "r"(body * 4), "r"(smem_u32(bar))
                   : "memory");
    }
    if (lane < head || (lane >= 4 && lane - 4 < tail)) dst[lane < 4 ? lane : head + body + lane - 4] = word;
  }
};

__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

// Whether `yes` holds for every worker.
__device__ __forceinline__ bool workers_all(bool yes) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)yes), "n"(kWorkers)
      : "memory");
  return all != 0;
}

template <bool VEC>
__global__ void __launch_bounds__(kWorkers + 32, 1)
    k_logit_rules_stream(const __grid_constant__ RuleArgs a, int rows, int slices, int slice, uint32_t slice_mul) {
  extern __shared__ char smem_raw[];
  RuleShared& sh = *reinterpret_cast<RuleShared*>(smem_raw + (128 - (smem_u32(smem_raw) & 127)) % 128);
  const int tid = threadIdx.x, lane = tid & 31, V = a.vocab;
  const long items = (long)rows * slices;
  const bool sort = slices > 1 && slices <= kSorted;
  const long first = items * blockIdx.x / gridDim.x, last = items * (blockIdx.x + 1) / gridDim.x;
  if (tid < kRing) {
    mbar_init(&sh.full[tid], 1);
    mbar_init(&sh.empty[tid], 1);
  }
  if (tid < 2) sh.n_list[tid] = 0;
  for (int e = tid; e < kMostIds; e += kWorkers + 32) sh.cnt[e] = 0;
  mbar_fence_init();
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  if (tid >= kWorkers) {
    RuleSlice s;
    s.row = -1;
    for (long it = first; it < last; it++) {
      const int k = (int)(it - first), at = k % kRing;
      RuleStage& st = sh.ring[at];
      const int row = (int)(it / slices);
      const float* in = a.in + (size_t)row * a.ld;
      const bool fresh = row != s.row;
      if (fresh) {
        s.row = row;
        s.i0 = s.i1 = s.b0 = s.b1 = 0;
        s.made = 0xFFFFFFFFu;
        if (a.r.tokens) {
          s.i0 = a.r.token_start[row];
          s.i1 = max(s.i0, a.r.token_start[row + 1]);
          if (a.r.generated_start) s.made = a.r.generated_start[row];
        }
        if (a.r.bias_ids) {
          s.b0 = a.r.bias_start[row];
          s.b1 = max(s.b0, a.r.bias_start[row + 1]);
        }
        s.w.rep = a.r.repetition ? a.r.repetition[row] : 1.f;
        s.w.freq = a.r.frequency ? a.r.frequency[row] : 0.f;
        s.w.pres = a.r.presence ? a.r.presence[row] : 0.f;
        s.masked = -1;
        if (a.r.mask) {
          const uint32_t m = a.r.mask_row ? a.r.mask_row[row] : (uint32_t)row;
          if (m < (uint32_t)a.r.n_masks)
            s.masked = (int)m;
          else if (m != kNoMask && lane == 0)
            atomicExch(&a.flags[FLAG_RANGE], RANGE_RULE);
        }
      }
      s.s0 = (int)(it - (long)row * slices) * slice - (VEC ? (int)skew_of(in) : 0);
      const int id0 = max(s.s0, 0), id1 = min(s.s0 + slice, V);
      s.word0 = id0 >> 5;
      Bring x, tok, ids, val, msk;
      x.head = x.body = x.tail = tok.head = tok.body = tok.tail = ids.head = ids.body = ids.tail = 0;
      val.head = val.body = val.tail = msk.head = msk.body = msk.tail = 0;
      if (id1 > id0) {
        // with !VEC a slice may begin anywhere: positions keep the distance to a 16-byte boundary
        x.ask(st.x + (VEC ? id0 - s.s0 : skew_of(in + id0)), in + id0, id1 - id0, lane);
        if (s.i1 > s.i0 && (fresh || !sort))
          tok.ask(st.tokens + skew_of(a.r.tokens + s.i0), a.r.tokens + s.i0, min(s.i1 - s.i0, (uint32_t)kTokenRoom), lane);
        if (s.b1 > s.b0) {
          const uint32_t n = min(s.b1 - s.b0, (uint32_t)kBiasRoom);
          ids.ask(st.bias_ids + skew_of(a.r.bias_ids + s.b0), a.r.bias_ids + s.b0, n, lane);
          val.ask(st.bias + skew_of(a.r.bias + s.b0), a.r.bias + s.b0, n, lane);
        }
        if (s.masked >= 0) {
          const uint32_t* m = a.r.mask + (size_t)s.masked * ((V + 31) / 32) + s.word0;
          msk.ask(st.mask + skew_of(m), m, ((id1 - 1) >> 5) - s.word0 + 1, lane);
        }
      }
      if (k >= kRing && !mbar_wait(&sh.empty[at], (k / kRing - 1) & 1, a.flags, kWaitSite)) break;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      x.put(&sh.full[at], lane);
      tok.put(&sh.full[at], lane);
      ids.put(&sh.full[at], lane);
      val.put(&sh.full[at], lane);
      msk.put(&sh.full[at], lane);
      if (lane == 0) st.s = s;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.full[at]);
    }
    return;
  }

  bool bad = false;
  int turn = 0;  // slices of rows with ids so far
  int sorted_row = -1, checked_row = -1, wild_row = -1;  // wild: its bias ids do not increase
  for (long it = first; it < last; it++) {
    const int k = (int)(it - first), at = k % kRing;
    RuleStage& st = sh.ring[at];
    // a wait that ran out is reported; what the stage then holds is not looked at
    if (!workers_all(mbar_wait(&sh.full[at], (k / kRing) & 1, a.flags, kWaitSite))) break;
    const RuleSlice s = st.s;  // in registers: shared memory is written all the time below
    const int s0 = s.s0, id0 = max(s0, 0), id1 = min(s0 + slice, V);
    if (id1 > id0) {
      float* x = st.x + (VEC ? 0 : (int)skew_of(a.in + (size_t)s.row * a.ld + id0));  // position e = id - s0
      const uint32_t n_tok = s.i1 - s.i0, span = id1 - id0;
      if (n_tok) {
        const uint32_t skew = skew_of(a.r.tokens + s.i0), here = min(n_tok, (uint32_t)kTokenRoom);
        const uint32_t made = s.made > s.i0 ? s.made - s.i0 : 0;
        uint32_t most = 0;
        auto count = [&](bool gen, uint32_t id) {
          most = max(most, id);
          if (id - (uint32_t)id0 < span) {
            const uint32_t p = id - (uint32_t)s0;
            uint32_t old;
            if (gen)
              old = atomicAdd(&sh.cnt[p], 1u);
            else
              old = atomicOr(&sh.cnt[p], kSeen);
            if (old == 0) sh.list[atomicAdd(&sh.n_list[turn & 1], 1u)] = (uint16_t)p;
          }
        };
        if (sort) {
          const int bin = (int)(it - (long)s.row * slices);
          if (s.row != sorted_row) {
            sorted_row = s.row;
            const uint32_t lead = (uint32_t)(bin * slice - s0);
            constexpr int PER = (kTokenRoom + kWorkers - 1) / kWorkers;
            uint32_t mine[PER], rank[PER];
            if (tid <= kSorted) sh.bins[tid] = 0;
            workers_sync();
#pragma unroll
            for (int j = 0; j < PER; j++) {
              const uint32_t i = j * kWorkers + tid;
              if (j * kWorkers >= here) break;
              const uint32_t id = i < here ? st.tokens[skew + i] : 0xFFFFFFFFu;
              if (i < here) most = max(most, id);
              const uint32_t to = id < (uint32_t)V ? __umulhi(id + lead, slice_mul) : kSorted;
              const uint32_t same = __match_any_sync(0xffffffffu, to);
              const int leader = __ffs(same) - 1;
              uint32_t base = 0;
              if (lane == leader && to < kSorted) base = atomicAdd(&sh.bins[to], (uint32_t)__popc(same));
              rank[j] = __shfl_sync(0xffffffffu, base, leader) + __popc(same & ((1u << lane) - 1));
              mine[j] = to < kSorted ? id | (i >= made ? kSeen : 0) : 0xFFFFFFFFu;
            }
            workers_sync();
            if (tid < 32) {  // where each slice's ids begin
              const uint32_t c0 = sh.bins[2 * lane], c1 = sh.bins[2 * lane + 1];
              uint32_t sum = c0 + c1;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
              }
              sh.bins[2 * lane] = sum - c0 - c1;
              sh.bins[2 * lane + 1] = sum - c1;
              if (lane == 31) sh.bins[kSorted] = sum;
            }
            workers_sync();
#pragma unroll
            for (int j = 0; j < PER; j++) {
              if (j * kWorkers >= here) break;
              if (mine[j] != 0xFFFFFFFFu) sh.sorted[sh.bins[__umulhi((mine[j] & ~kSeen) + lead, slice_mul)] + rank[j]] = mine[j];
            }
            workers_sync();
          }
          // the warp's new ids take their places in the list with one atomic
          const uint32_t end = sh.bins[bin + 1];
          for (uint32_t i0 = sh.bins[bin] + (tid & ~31); i0 < end; i0 += kWorkers) {
            uint32_t p = 0;
            bool fresh = false;
            if (i0 + lane < end) {
              const uint32_t y = sh.sorted[i0 + lane];
              p = (y & ~kSeen) - (uint32_t)s0;
              fresh = ((y & kSeen) ? atomicAdd(&sh.cnt[p], 1u) : atomicOr(&sh.cnt[p], kSeen)) == 0;
            }
            const uint32_t all = __ballot_sync(0xffffffffu, fresh);
            uint32_t at = 0;
            if (lane == 0 && all) at = atomicAdd(&sh.n_list[turn & 1], (uint32_t)__popc(all));
            at = __shfl_sync(0xffffffffu, at, 0);
            if (fresh) sh.list[at + __popc(all & ((1u << lane) - 1))] = (uint16_t)p;
          }
        } else {
          for (uint32_t q = tid * 4; q < here + skew; q += kWorkers * 4) {  // ids q - skew .. + 3
            const uint4 u = *reinterpret_cast<const uint4*>(st.tokens + q);
            if (q >= skew && q + 4 <= here + skew) {
              count(q - skew >= made, u.x);
              count(q + 1 - skew >= made, u.y);
              count(q + 2 - skew >= made, u.z);
              count(q + 3 - skew >= made, u.w);
            } else {
              if (q >= skew) count(q - skew >= made, u.x);
              if (q + 1 >= skew && q + 1 < here + skew) count(q + 1 - skew >= made, u.y);
              if (q + 2 >= skew && q + 2 < here + skew) count(q + 2 - skew >= made, u.z);
              if (q + 3 >= skew && q + 3 < here + skew) count(q + 3 - skew >= made, u.w);
            }
          }
        }
        for (uint32_t i = here + tid; i < n_tok; i += kWorkers) count(i >= made, a.r.tokens[s.i0 + i]);
        bad |= most >= (uint32_t)V;
      }
      const uint32_t* ids = st.bias_ids + skew_of(a.r.bias_ids + s.b0);
      const float* val = st.bias + skew_of(a.r.bias + s.b0);
      uint32_t n_bias = s.b1 - s.b0;
      const uint32_t n_here = min(n_bias, (uint32_t)kBiasRoom);
      auto bias_id = [&](uint32_t i) { return i < n_here ? ids[i] : a.r.bias_ids[s.b0 + i]; };
      if (n_bias && s.row != checked_row) {
        // an id that comes twice would belong to two threads: such a row takes none of its biases
        checked_row = s.row;
        bool wild = false;
        for (uint32_t i = tid + 1; i < n_bias; i += kWorkers) wild |= bias_id(i - 1) >= bias_id(i);
        if (!workers_all(!wild)) {
          bad = true;
          wild_row = s.row;
        }
      }
      if (s.row == wild_row) n_bias = 0;
      // (biases go to the last warps first, ids to the first: few of either keep different warps busy)
      for (uint32_t i = kWorkers - 1 - tid; i < n_bias; i += kWorkers) {
        const uint32_t id = bias_id(i);
        bad |= id >= (uint32_t)V;
        if (id - (uint32_t)id0 < span) atomicOr(&sh.cnt[id - (uint32_t)s0], kBiased);
      }
      if (n_tok || n_bias) {
        workers_sync();
        // ids with a bias belong to it, the others to the list
        for (uint32_t i = kWorkers - 1 - tid; i < n_bias; i += kWorkers) {
          const uint32_t id = bias_id(i), p = id - (uint32_t)s0;
          if (id - (uint32_t)id0 < span) {
            x[p] = penalise(s.w, x[p], sh.cnt[p]) + (i < n_here ? val[i] : a.r.bias[s.b0 + i]);
            sh.cnt[p] = 0;
          }
        }
        const uint32_t n = sh.n_list[turn & 1];
        for (uint32_t i = tid; i < n; i += kWorkers) {
          const uint32_t p = sh.list[i], c = sh.cnt[p];
          if (c != 0 && !(c & kBiased)) {
            x[p] = penalise(s.w, x[p], c);
            sh.cnt[p] = 0;
          }
        }
        turn++;
        if (tid == 0) sh.n_list[turn & 1] = 0;
        workers_sync();
      }
      const bool masked = s.masked >= 0;
      const uint32_t* mask =
          masked ? st.mask + skew_of(a.r.mask + (size_t)s.masked * ((V + 31) / 32) + s.word0) : nullptr;
      const uint32_t words = ((id1 - 1) >> 5) - s.word0 + 1;
      if (VEC) {
        if (masked) {
          constexpr int TURNS = (kMostIds + kWorkers * 4 - 1) / (kWorkers * 4);
          uint32_t open[TURNS];
#pragma unroll
          for (int k = 0; k < TURNS; k++) {
            const int e = (k * kWorkers + tid) * 4, id = s0 + e, from = max(id, 0);
            open[k] = 0xF;
            if (e < slice && id < id1) {
              const uint32_t wd = (from >> 5) - s.word0, low = mask[wd], high = wd + 1 < words ? mask[wd + 1] : 0;
              open[k] = __funnelshift_r(low, high, from & 31) << (from - id);
            }
          }
#pragma unroll
          for (int k = 0; k < TURNS; k++) {
            if ((open[k] & 0xF) == 0xF) continue;
            float4* at = reinterpret_cast<float4*>(x + (k * kWorkers + tid) * 4);
            float4 y = *at;
            if (!(open[k] & 1)) y.x = -INFINITY;
            if (!(open[k] & 2)) y.y = -INFINITY;
            if (!(open[k] & 4)) y.z = -INFINITY;
            if (!(open[k] & 8)) y.w = -INFINITY;
            *at = y;
          }
        }
      } else {
        float* out = a.out + (size_t)s.row * a.out_ld;
        for (int id = id0 + tid; id < id1; id += kWorkers) {
          float y = x[id - s0];
          if (masked && !((mask[(id >> 5) - s.word0] >> (id & 31)) & 1)) y = -INFINITY;
          out[id] = y;
        }
      }
    }
    // what was written here goes out by a bulk store (VEC), or comes in by the next bulk copy
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    workers_sync();
    if (VEC) {
      // The stage is free once the store has read it: when the next one is on its way.
      if (id1 > id0) {
        float* out = a.out + (size_t)s.row * a.out_ld + id0;
        const float* x = st.x + (id0 - s0);
        const uint32_t n = id1 - id0, head = min((4 - skew_of(out)) & 3, n), body = (n - head) & ~3u, tail = n - head - body;
        if (tid == 0 && body)
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(out + head),
                       "r"(smem_u32(x + head)), "r"(body * 4)
                       : "memory");
        if (lane < head && tid < 32) out[lane] = x[lane];
        if (tid >= 32 && tid - 32 < tail) out[head + body + lane] = x[head + body + lane];
      }
      if (tid == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      if (k > 0) {
        if (tid == 0) {
          asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          mbar_arrive(&sh.empty[(k - 1) % kRing]);
        }
      }
      __syncwarp();
    } else if (tid == 0) {
      mbar_arrive(&sh.empty[at]);
    }
  }
  if (VEC && tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  if (bad) atomicExch(&a.flags[FLAG_RANGE], RANGE_RULE);
}

// How a row is cut: the number of slices (of kMostIds at most) that gives the fullest last turn.
int rules_stream(turt_ctx* ctx, const RuleArgs& a, int rows, bool vec) {
  static std::atomic<uint64_t> done{0}, done_vec{0};
  int sms = 0;
  RC(sm_count(ctx->device, &sms));
  const int extra = vec ? 3 : 0, least = ceil_div((long)a.vocab + extra, kMostIds - 4);
  int slices = least, slice = 0;
  long best = 0;
  for (int n = least; n <= 2 * least + 2; n++) {
    const int len = (ceil_div((long)a.vocab + extra, n) + 3) & ~3;
    const long cost = (long)ceil_div((long)rows * n, sms) * (len + 512);  // 512: what a slice costs besides its ids
    if (slice == 0 || cost < best) {
      best = cost;
      slices = n;
      slice = len;
    }
  }
  slices = ceil_div((long)a.vocab + extra, slice);
  static_assert(sizeof(RuleShared) + 128 <= 227 * 1024, "shared memory");
  const int smem = (int)sizeof(RuleShared) + 128, grid = (int)std::min((long)rows * slices, (long)sms);
  auto kern = vec ? k_logit_rules_stream<true> : k_logit_rules_stream<false>;
  RC(smem_attr_per_device(vec ? done_vec : done, kern, smem));
  TURT_CHECK_CUDA(launch_pdl(kern, dim3(grid), dim3(kWorkers + 32), smem, ctx->stream, a, rows, slices, slice,
                             (uint32_t)(((1ull << 32) + slice - 1) / slice)));
  TURT_LAUNCH_CHECK();
  return OK;
}

}  // namespace
}  // namespace turt

using namespace turt;

extern "C" int turt_logit_rules_apply(turt_ctx* ctx, const float* logits, size_t ld, float* out, size_t out_ld,
                                      int rows, int vocab, const turt_logit_rules* rules) {
  TURT_REQUIRE(rules, "logit_rules: null rules");
  TURT_REQUIRE(rows >= 0 && vocab >= 0 && vocab <= 0x7fff0000, "logit_rules: bad size");
  TURT_REQUIRE(rows <= 65535, "logit_rules: at most 65535 rows");
  const turt_logit_rules& r = *rules;
  TURT_REQUIRE(!r.tokens || r.token_start, "logit_rules: tokens need token_start");
  TURT_REQUIRE(r.tokens || !(r.repetition || r.frequency || r.presence || r.generated_start),
               "logit_rules: penalties need tokens");
  TURT_REQUIRE(!r.bias_ids || (r.bias && r.bias_start), "logit_rules: bias_ids need bias and bias_start");
  TURT_REQUIRE(!r.mask || r.n_masks > 0, "logit_rules: masks need n_masks");
  TURT_REQUIRE(!r.mask || r.mask_row || r.n_masks >= rows, "logit_rules: without mask_row there is a mask per row");
  TURT_REQUIRE(rows == 0 || vocab == 0 || (logits && out), "logit_rules: null pointer");
  TURT_REQUIRE(rows <= 1 || (ld >= (size_t)vocab && out_ld >= (size_t)vocab), "logit_rules: pitch below vocab");
  TURT_REQUIRE(out != logits || ld == out_ld, "logit_rules: working in place needs equal pitches");
  TURT_REQUIRE(((uintptr_t)logits | (uintptr_t)out | (uintptr_t)r.tokens | (uintptr_t)r.token_start |
                (uintptr_t)r.generated_start | (uintptr_t)r.repetition | (uintptr_t)r.frequency | (uintptr_t)r.presence |
                (uintptr_t)r.bias_ids | (uintptr_t)r.bias | (uintptr_t)r.bias_start | (uintptr_t)r.mask |
                (uintptr_t)r.mask_row) % 4 == 0,
               "logit_rules: misaligned pointer");
  TURT_REQUIRE(ctx, "null context");
  TURT_CHECK_CUDA(cudaSetDevice(ctx->device));
  if (rows == 0 || vocab == 0) return OK;
  RuleArgs a;
  a.r = r;
  a.in = logits, a.out = out;
  a.ld = ld, a.out_ld = out_ld;
  a.vocab = vocab;
  a.flags = ctx->flags;
  // every row of in and out starts equally far from a 16-byte boundary
  const bool vec = ((uintptr_t)logits & 15) == ((uintptr_t)out & 15) && (rows == 1 || ld % 4 == out_ld % 4);
  // The pipeline where every SM gets several slices (256 x 128000: 69 us, one block per slice 100 us; but
  // 64 x 50001: 11.5 us, one block per slice 9.5 us); short slices where even those would leave SMs idle
  // (1 x 8192: 3.2 us, slices of 4096 4.0 us; 64 x 50001: 12.3 us, slices of 4096 9.5 us).
  const long enough = 4 * 148;
  if (rows * (long)ceil_div(vocab, kMostIds) >= enough) return rules_stream(ctx, a, rows, vec);
  if (rows * (long)ceil_div(vocab, 4096) >= enough) return rules_launch<256, 4>(ctx->stream, a, rows, vec);
  return rules_launch<128, 2>(ctx->stream, a, rows, vec);
}
