// rules.cu -- per-request rules on the logits of the next token: penalties for repeated tokens,
// biases and grammar masks.
//
//   n = times that id v was generated in row r;  seen = v in the prompt or generated
//   x = logits;  seen: x = x > 0 ? x / rep : x * rep;  n > 0: x -= freq * n, x -= pres;
//   x += bias[v];  mask bit 0: x = -infinity
//
// One pass over the logits: a block owns a slice of one row's vocabulary, counts the row's ids that
// fall into the slice in shared memory (integer atomics: the counts do not depend on their order)
// and applies everything while the slice streams through.
#include "../../include/turt_cuda.h"
#include "ctx.cuh"

namespace turt {
namespace {

constexpr int kRuleThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;  // count word: bit 31 = in the prompt, the rest = times generated
constexpr uint32_t kNoMask = 0xFFFFFFFFu;

struct RuleArgs {
  turt_logit_rules r;
  const float* in;
  float* out;
  size_t ld, out_ld;
  int vocab, slice;
  int* flags;
};

struct RowRules {
  float rep, freq, pres;
  const uint32_t* mask;
};

__device__ __forceinline__ float apply_rules(const RowRules& w, float x, uint32_t c, float bias, bool open) {
  if (c) {
    x = x > 0.f ? x / w.rep : x * w.rep;
    const uint32_t n = c & ~kSeen;
    if (n) {
      x -= w.freq * (float)n;
      x -= w.pres;
    }
  }
  x += bias;
  return open ? x : -INFINITY;
}

// Slices are cut where a float4 of the row starts: `lead` elements lie between that boundary and the row's
// first, so position e of the slice's arrays is id e - lead.  VEC: 16-byte loads and stores.
template <bool VEC>
__global__ void __launch_bounds__(kRuleThreads) k_logit_rules(const __grid_constant__ RuleArgs a) {
  extern __shared__ __align__(16) uint32_t cnt[];  // [slice] counts, [slice] biases
  float* bias = reinterpret_cast<float*>(cnt + a.slice);
  const int r = blockIdx.y, V = a.vocab;
  const float* in = a.in + (size_t)r * a.ld;
  float* out = a.out + (size_t)r * a.out_ld;
  const int lead = VEC ? (int)((reinterpret_cast<uintptr_t>(in) >> 2) & 3) : 0;
  const int s0 = blockIdx.x * a.slice - lead;  // id of the slice's first position (may be negative)
  const bool first = blockIdx.x == 0;
  if (s0 >= V) return;
  pdl_wait();
  pdl_trigger();
  const bool hist = a.r.tokens != nullptr, biased = a.r.bias_ids != nullptr;
  if (hist)
    for (int e = threadIdx.x * 4; e < a.slice; e += kRuleThreads * 4) *reinterpret_cast<uint4*>(cnt + e) = make_uint4(0, 0, 0, 0);
  if (biased)
    for (int e = threadIdx.x * 4; e < a.slice; e += kRuleThreads * 4)
      *reinterpret_cast<float4*>(bias + e) = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  bool bad = false;
  if (hist) {
    const uint32_t i1 = a.r.token_start[r + 1], g = a.r.generated_start ? a.r.generated_start[r] : 0xFFFFFFFFu;
    for (uint32_t i = a.r.token_start[r] + threadIdx.x; i < i1; i += kRuleThreads) {
      const uint32_t id = a.r.tokens[i];
      const uint32_t e = id - (uint32_t)s0;
      if (id >= (uint32_t)V)
        bad = true;
      else if (e < (uint32_t)a.slice) {
        if (i >= g)
          atomicAdd(&cnt[e], 1u);
        else
          atomicOr(&cnt[e], kSeen);
      }
    }
  }
  if (biased) {
    const uint32_t i0 = a.r.bias_start[r], i1 = a.r.bias_start[r + 1];
    for (uint32_t i = i0 + threadIdx.x; i < i1; i += kRuleThreads) {
      const uint32_t id = a.r.bias_ids[i];
      const uint32_t e = id - (uint32_t)s0;
      if (id >= (uint32_t)V || (first && i > i0 && a.r.bias_ids[i - 1] >= id))
        bad = true;
      else if (e < (uint32_t)a.slice)
        bias[e] = a.r.bias[i];
    }
  }
  RowRules w;
  w.rep = a.r.repetition ? a.r.repetition[r] : 1.f;
  w.freq = a.r.frequency ? a.r.frequency[r] : 0.f;
  w.pres = a.r.presence ? a.r.presence[r] : 0.f;
  w.mask = nullptr;
  if (a.r.mask) {
    const uint32_t m = a.r.mask_row ? a.r.mask_row[r] : (uint32_t)r;
    if (m < (uint32_t)a.r.n_masks)
      w.mask = a.r.mask + (size_t)m * ((V + 31) / 32);
    else if (m != kNoMask)
      bad = true;
  }
  if (bad) atomicExch(&a.flags[FLAG_RANGE], RANGE_RULE);
  __syncthreads();
  if (VEC) {
    for (int e = threadIdx.x * 4; e < a.slice; e += kRuleThreads * 4) {
      const int id = s0 + e;
      if (id >= V) break;
      uint4 c = hist ? *reinterpret_cast<uint4*>(cnt + e) : make_uint4(0, 0, 0, 0);
      float4 bs = biased ? *reinterpret_cast<float4*>(bias + e) : make_float4(0.f, 0.f, 0.f, 0.f);
      uint32_t open = 0xF;
      if (w.mask) {
        open = 0;
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (id + j >= 0 && id + j < V) open |= ((w.mask[(id + j) >> 5] >> ((id + j) & 31)) & 1) << j;
      }
      if (id >= 0 && id + 4 <= V) {
        float4 x = *reinterpret_cast<const float4*>(in + id);
        x.x = apply_rules(w, x.x, c.x, bs.x, open & 1);
        x.y = apply_rules(w, x.y, c.y, bs.y, open & 2);
        x.z = apply_rules(w, x.z, c.z, bs.z, open & 4);
        x.w = apply_rules(w, x.w, c.w, bs.w, open & 8);
        *reinterpret_cast<float4*>(out + id) = x;
      } else {
        const uint32_t cc[4] = {c.x, c.y, c.z, c.w};
        const float bb[4] = {bs.x, bs.y, bs.z, bs.w};
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (id + j >= 0 && id + j < V) out[id + j] = apply_rules(w, in[id + j], cc[j], bb[j], (open >> j) & 1);
      }
    }
  } else {
    for (int e = threadIdx.x; e < a.slice; e += kRuleThreads) {
      const int id = s0 + e;
      if (id >= V) break;
      const bool open = !w.mask || ((w.mask[id >> 5] >> (id & 31)) & 1);
      out[id] = apply_rules(w, in[id], hist ? cnt[e] : 0, biased ? bias[e] : 0.f, open);
    }
  }
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
  TURT_REQUIRE(((uintptr_t)logits | (uintptr_t)out) % 4 == 0, "logit_rules: misaligned pointer");
  TURT_REQUIRE(ctx, "null context");
  TURT_CHECK_CUDA(cudaSetDevice(ctx->device));
  if (rows == 0 || vocab == 0) return OK;
  RuleArgs a;
  a.r = r;
  a.in = logits, a.out = out;
  a.ld = ld, a.out_ld = out_ld;
  a.vocab = vocab;
  a.flags = ctx->flags;
  a.slice = 4096;
  // every row of in and out starts equally far from a 16-byte boundary
  const bool vec = ((uintptr_t)logits & 15) == ((uintptr_t)out & 15) && (rows == 1 || ld % 4 == out_ld % 4);
  const size_t smem = (size_t)a.slice * 8;
  const dim3 grid(ceil_div((long)vocab + 3, a.slice), rows);
  TURT_CHECK_CUDA(launch_pdl(vec ? k_logit_rules<true> : k_logit_rules<false>, grid, dim3(kRuleThreads), smem, ctx->stream, a));
  TURT_LAUNCH_CHECK();
  return OK;
}
