// scores_abi.hip — the C-ABI entries of the token scores and the top-k
// distillation (k_scores.hip). They allocate nothing and share nothing:
// scratch is the caller's, so calls on several streams and captured graphs
// need only scratch of their own. Every argument is checked here, before any
// launch; what lies in device memory (ids, values) is checked by the kernels.
#include <hip/hip_runtime.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "abi_checks.h"

namespace seeml_hip {
namespace {

static_assert(kF32 == SEEML_HIP_F32 && kBF16 == SEEML_HIP_BF16 && kF16 == SEEML_HIP_F16);
static_assert(kTopkMax == SEEML_HIP_TOPK_MAX && kScoreStats == SEEML_HIP_TOKEN_STATS &&
              kDistillStats == SEEML_HIP_DISTILL_STATS);

// A launch has fewer than 2^32 threads: a workgroup of at most 1024 for each
// row, and in the gradients one of 256 for each row and 16 KiB. Classes are
// counted in 30 bits.
constexpr uint64_t kMaxRows = (uint64_t{1} << 22) - 1;
constexpr uint64_t kMaxClasses = uint64_t{1} << 30;
constexpr uint64_t kMaxBytes = uint64_t{1} << 37;

struct Call : AbiCall {
  Status Shape(int dtype, uint64_t N, uint64_t C, uint64_t stride, uint64_t k, double T) const {
    if (dtype != kF32 && dtype != kBF16 && dtype != kF16)
      return Fail("unknown logits type " + std::to_string(dtype));
    if (N == 0 || C == 0) return Fail("empty input");
    if (N > kMaxRows) return Fail("too many rows");
    if (C > kMaxClasses) return Fail("too many classes");
    if (N * C > kMaxBytes / ElemSize(dtype)) return Fail("more than 2^37 bytes of logits");
    if (stride < C) return Fail("row stride below the number of classes");
    uint64_t bytes = 0;
    if (!MulOk(stride, N * ElemSize(dtype), &bytes) || bytes >= uint64_t{1} << 62)
      return Fail("row stride too large");
    if (k > kTopkMax) return Fail("more than " + std::to_string(kTopkMax) + " listed classes");
    if (k > C) return Fail("more listed classes than classes");
    if (!(T >= 1e-30 && T <= 1e30)) return Fail("temperature outside 1e-30 .. 1e30");
    return Status::Ok();
  }

  // dlogits is the logits (same rows, in place), other columns of the same
  // rows, or elsewhere.
  Status GradientPlace(const void* x, uint64_t stride, const void* dx, uint64_t dstride, uint64_t N,
                       uint64_t C, size_t es) const {
    if (dstride < C) return Fail("gradient row stride below the number of classes");
    uint64_t bytes = 0;
    if (!MulOk(dstride, N * es, &bytes) || bytes >= uint64_t{1} << 62)
      return Fail("gradient row stride too large");
    if (x == dx) {
      if (stride != dstride && N > 1)
        return Fail("dlogits overlaps logits with another row stride");
      return Status::Ok();
    }
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(dx);
    const uint64_t ab = ((N - 1) * stride + C) * es, bb = ((N - 1) * dstride + C) * es;
    if (a >= b + bb || b >= a + ab) return Status::Ok();
    if (stride == dstride) {
      const uint64_t row = stride * es, row_bytes = C * es;
      const uint64_t gap = b > a ? (b - a) % row : (row - (a - b) % row) % row;
      if (gap >= row_bytes && gap + row_bytes <= row) return Status::Ok();
    }
    return Fail("dlogits overlaps logits");
  }
};

// What the three distillation entries share.
Status CheckDistill(const Call& call, const TopkDistillArgs& a, uint64_t k, uint64_t scratch_bytes,
                    bool fwd, bool bwd, bool scratch) {
  if (Status s = call.Shape(a.dtype, a.N, a.C, a.stride, k, a.T); !s) return s;
  if (k == 0) return call.Fail("no listed classes");
  if (!a.logits || !a.t_ids || !a.t_logp) return call.Fail("null logits, t_ids or t_logp");
  if (fwd && !a.row_loss) return call.Fail("null row_loss");
  if (bwd && !a.dlogits) return call.Fail("null dlogits");
  if (bwd && !fwd && !a.stats) return call.Fail("null row_stats");
  if (a.tail != 0 && a.tail != 1) return call.Fail("tail is 0 or 1");
  const size_t es = ElemSize(a.dtype);
  if (bwd)
    if (Status s = call.GradientPlace(a.logits, a.stride, a.dlogits, a.dstride, a.N, a.C, es); !s)
      return s;
  const uint64_t need = scratch ? TopkDistillScratch(a.N, a.C, a.dtype, k) : 0;
  if (Status s = call.Scratch(a.scratch, scratch_bytes, need); !s) return s;
  const uint64_t xb = ((a.N - 1) * a.stride + a.C) * es;
  const Span ids{"t_ids", a.t_ids, a.N * k * 4, false, 4};
  const Span lps{"t_logp", a.t_logp, a.N * k * 4, false, 4};
  const Span wts{"row_weight", a.weight, a.N * 4, false, 4};
  const Span seed{"seed", bwd ? a.seed : nullptr, 4, false, 4};
  const Span loss{"loss", fwd ? a.loss : nullptr, 4, true, 4};
  const Span rows{"row_loss", fwd ? a.row_loss : nullptr, a.N * 4, true, 4};
  const Span stats{"row_stats", a.stats, a.N * kDistillStats * 4, fwd, 4};
  const Span scr{"scratch", need ? a.scratch : nullptr, need, true, 16};
  if (Status s = call.Ranges({{"logits", a.logits, xb, false, es}, ids, lps, wts, seed, loss, rows,
                              stats, scr});
      !s)
    return s;
  if (bwd) {  // dlogits against everything but the logits, which it may be
    const uint64_t db = ((a.N - 1) * a.dstride + a.C) * es;
    if (Status s = call.Ranges({{"dlogits", a.dlogits, db, true, es}, ids, lps, wts, seed, loss,
                                rows, stats, scr});
        !s)
      return s;
  }
  return Status::Ok();
}

}  // namespace
}  // namespace seeml_hip

using namespace seeml_hip;

extern "C" {

uint64_t seeml_hip_token_logprobs_scratch(uint64_t N, uint64_t C, int dtype, uint64_t k) {
  const Call call{{"TokenLogprobs"}};
  return call.Shape(dtype, N, C, C, k, 1.0) ? TokenScoreScratch(N, C, dtype, k) : 0;
}

int seeml_hip_token_logprobs_fwd(const void* logits, int dtype, uint64_t row_stride,
                                 const int32_t* targets, double T, uint64_t k, float* logp,
                                 float* entropy, float* row_stats, int32_t* top_ids,
                                 float* top_logp, uint64_t N, uint64_t C, void* scratch,
                                 uint64_t scratch_bytes, void* stream) {
  return Entry([&]() -> Status {
    const Call call{{"TokenLogprobs"}};
    if (Status s = call.Shape(dtype, N, C, row_stride, k, T); !s) return s;
    if (!logits) return call.Fail("null logits");
    if (!targets != !logp) return call.Fail("targets and logp go together");
    if (k > 0 && (!top_ids || !top_logp)) return call.Fail("null top_ids or top_logp");
    if (!logp && !entropy && !row_stats && k == 0) return call.Fail("no output");
    const uint64_t need = TokenScoreScratch(N, C, dtype, k);
    if (Status s = call.Scratch(scratch, scratch_bytes, need); !s) return s;
    const size_t es = ElemSize(dtype);
    if (Status s = call.Ranges({{"logits", logits, ((N - 1) * row_stride + C) * es, false, es},
                                {"targets", targets, N * 4, false, 4},
                                {"logp", logp, N * 4, true, 4},
                                {"entropy", entropy, N * 4, true, 4},
                                {"row_stats", row_stats, N * kScoreStats * 4, true, 4},
                                {"top_ids", k ? top_ids : nullptr, N * k * 4, true, 4},
                                {"top_logp", k ? top_logp : nullptr, N * k * 4, true, 4},
                                {"scratch", need ? scratch : nullptr, need, true, 16}});
        !s)
      return s;
    if (Status s = call.OnDevice(logits, stream, "logits"); !s) return s;
    return TokenScoreFwd({logits, dtype, row_stride, targets, T, static_cast<uint32_t>(k), logp,
                          entropy, row_stats, top_ids, top_logp, N, C, scratch},
                         On(stream));
  });
}

int seeml_hip_token_logprobs_bwd(const void* logits, int dtype, uint64_t row_stride,
                                 const int32_t* targets, double T, const float* row_stats,
                                 const float* dlogp, const float* dentropy, void* dlogits,
                                 uint64_t dlogits_stride, uint64_t N, uint64_t C, void* stream) {
  return Entry([&]() -> Status {
    const Call call{{"TokenLogprobsBwd"}};
    if (Status s = call.Shape(dtype, N, C, row_stride, 0, T); !s) return s;
    if (!logits || !row_stats || !dlogits) return call.Fail("null logits, row_stats or dlogits");
    if (!dlogp && !dentropy) return call.Fail("no gradient to carry back");
    if (dlogp && !targets) return call.Fail("dlogp without targets");
    const size_t es = ElemSize(dtype);
    if (Status s = call.GradientPlace(logits, row_stride, dlogits, dlogits_stride, N, C, es); !s)
      return s;
    if (Status s = call.Ranges({{"logits", logits, ((N - 1) * row_stride + C) * es, false, es}});
        !s)
      return s;
    if (Status s = call.Ranges({{"dlogits", dlogits, ((N - 1) * dlogits_stride + C) * es, true, es},
                                {"targets", targets, N * 4, false, 4},
                                {"row_stats", row_stats, N * kScoreStats * 4, false, 4},
                                {"dlogp", dlogp, N * 4, false, 4},
                                {"dentropy", dentropy, N * 4, false, 4}});
        !s)
      return s;
    if (Status s = call.OnDevice(logits, stream, "logits"); !s) return s;
    return TokenScoreBwd({logits, dtype, row_stride, dlogp ? targets : nullptr, T, row_stats,
                          dlogp, dentropy, dlogits, dlogits_stride, N, C},
                         On(stream));
  });
}

uint64_t seeml_hip_topk_distill_scratch(uint64_t N, uint64_t C, int dtype, uint64_t k) {
  const Call call{{"TopkDistill"}};
  return call.Shape(dtype, N, C, C, k, 1.0) ? TopkDistillScratch(N, C, dtype, k) : 0;
}

int seeml_hip_topk_distill_fwd(const void* logits, int dtype, uint64_t row_stride,
                               const int32_t* t_ids, const float* t_logp, uint64_t k,
                               const float* row_weight, double T, int tail, float* loss,
                               float* row_loss, float* row_stats, uint64_t N, uint64_t C,
                               void* scratch, uint64_t scratch_bytes, void* stream) {
  return Entry([&]() -> Status {
    const Call call{{"TopkDistill"}};
    const TopkDistillArgs a{logits, dtype, row_stride, t_ids, t_logp, static_cast<uint32_t>(k),
                            row_weight, nullptr, T, tail, loss, row_loss, row_stats, nullptr, 0, N,
                            C, scratch};
    if (Status s = CheckDistill(call, a, k, scratch_bytes, true, false, true); !s) return s;
    if (Status s = call.OnDevice(logits, stream, "logits"); !s) return s;
    return TopkDistillFwd(a, On(stream));
  });
}

int seeml_hip_topk_distill_bwd(const void* logits, int dtype, uint64_t row_stride,
                               const int32_t* t_ids, const float* t_logp, uint64_t k,
                               const float* row_weight, const float* seed, double T, int tail,
                               const float* row_stats, void* dlogits, uint64_t dlogits_stride,
                               uint64_t N, uint64_t C, void* stream) {
  return Entry([&]() -> Status {
    const Call call{{"TopkDistillBwd"}};
    const TopkDistillArgs a{logits, dtype, row_stride, t_ids, t_logp, static_cast<uint32_t>(k),
                            row_weight, seed, T, tail, nullptr, nullptr,
                            const_cast<float*>(row_stats), dlogits, dlogits_stride, N, C, nullptr};
    if (Status s = CheckDistill(call, a, k, 0, false, true, false); !s) return s;
    if (Status s = call.OnDevice(logits, stream, "logits"); !s) return s;
    return TopkDistillBwd(a, On(stream));
  });
}

int seeml_hip_topk_distill_fwd_bwd(const void* logits, int dtype, uint64_t row_stride,
                                   const int32_t* t_ids, const float* t_logp, uint64_t k,
                                   const float* row_weight, const float* seed, double T, int tail,
                                   float* loss, float* row_loss, void* dlogits,
                                   uint64_t dlogits_stride, uint64_t N, uint64_t C, void* scratch,
                                   uint64_t scratch_bytes, void* stream) {
  return Entry([&]() -> Status {
    const Call call{{"TopkDistill"}};
    const TopkDistillArgs a{logits, dtype, row_stride, t_ids, t_logp, static_cast<uint32_t>(k),
                            row_weight, seed, T, tail, loss, row_loss, nullptr, dlogits,
                            dlogits_stride, N, C, scratch};
    if (Status s = CheckDistill(call, a, k, scratch_bytes, true, true, true); !s) return s;
    if (Status s = call.OnDevice(logits, stream, "logits"); !s) return s;
    return TopkDistillFwdBwd(a, On(stream));
  });
}

}  // extern "C"
