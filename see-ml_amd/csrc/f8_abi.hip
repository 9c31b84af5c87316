// f8_abi.hip — the C-ABI entries of the block-scaled 8-bit operators (k_f8.hip,
// k_f8_gemm.hip, k_f8_lora.hip). They allocate nothing and share nothing: scratch is the
// caller's. Every argument is checked here, before any launch; codes and scales
// may hold any bytes.
#include "abi_checks.h"
#include "f8_format.h"

namespace seeml_hip {
namespace {

static_assert(f8::kBlock == SEEML_HIP_F8_BLOCK);

constexpr uint64_t kMaxExtent = uint64_t{1} << 24;
constexpr uint64_t kMaxValues = uint64_t{1} << 33;  // of a matrix, with its padding
constexpr uint64_t kMaxRank = SEEML_HIP_F8_RANK_MAX;

uint64_t CodesBytes(uint64_t rows, uint64_t cols) { return rows * f8::Up128(cols); }
uint64_t ScalesBytes(uint64_t rows, uint64_t cols) { return f8::Up128(cols) / f8::kBlock * f8::Up128(rows); }

struct F8Call : AbiCall {
  Status Extents(uint64_t rows, uint64_t cols) const {
    if (rows == 0 || cols == 0) return Fail("empty input");
    if (rows > kMaxExtent || cols > kMaxExtent) return Fail("more than 2^24 rows or columns");
    if (f8::Up128(rows) * f8::Up128(cols) >= kMaxValues) return Fail("2^33 values or more");
    return Status::Ok();
  }
  Status Type(int dtype) const {
    if (dtype != kF32 && dtype != kBF16 && dtype != kF16) return Fail("unknown type " + std::to_string(dtype));
    return Status::Ok();
  }
  Status Act(int act) const {
    if (act < 1 || act > 3) return Fail("unknown activation " + std::to_string(act));
    return Status::Ok();
  }
  Status Stride(const char* name, uint64_t stride, uint64_t rows, uint64_t cols, int dtype) const {
    if (stride < cols) return Fail(std::string(name) + " row stride below the row length");
    uint64_t bytes = 0;
    if (!MulOk(stride, rows * ElemSize(dtype), &bytes) || bytes >= uint64_t{1} << 62)
      return Fail(std::string(name) + " row stride too large");
    return Status::Ok();
  }
  // A gradient takes the place of what it is the gradient of (same rows), or
  // lies apart from it.
  Status InPlace(const Span& x, uint64_t stride, const Span& dx, uint64_t dstride, uint64_t rows) const {
    if (x.p == dx.p) {
      if (stride != dstride && rows > 1)
        return Fail(std::string(dx.name) + " overlaps " + x.name + " with another row stride");
      return Status::Ok();
    }
    if (x.lo() < dx.lo() + dx.bytes && dx.lo() < x.lo() + x.bytes)
      return Fail(std::string(dx.name) + " overlaps " + x.name);
    return Status::Ok();
  }
};

Span Rows(const char* name, const void* p, int dtype, uint64_t stride, uint64_t rows, uint64_t cols, bool write) {
  const size_t es = ElemSize(dtype);
  return {name, p, ((rows - 1) * stride + cols) * es, write, es};
}
Span Codes(const char* name, const uint8_t* p, uint64_t rows, uint64_t cols, bool write = false) {
  return {name, p, CodesBytes(rows, cols), write, 16};
}
Span Scales(const char* name, const uint8_t* p, uint64_t rows, uint64_t cols, bool write = false) {
  return {name, p, ScalesBytes(rows, cols), write, 16};
}

// A size, or 0 for extents that are refused.
template <typename Ok, typename F>
uint64_t SizeIf(Ok&& ok, F&& f) {
  try {
    return ok(F8Call{{""}}) ? f() : 0;
  } catch (...) {
    return 0;
  }
}

}  // namespace
}  // namespace seeml_hip

using namespace seeml_hip;

extern "C" {

uint64_t seeml_hip_f8_codes_bytes(uint64_t rows, uint64_t cols) {
  return SizeIf([&](const F8Call& c) { return static_cast<bool>(c.Extents(rows, cols)); },
                [&] { return CodesBytes(rows, cols); });
}
uint64_t seeml_hip_f8_scales_bytes(uint64_t rows, uint64_t cols) {
  return SizeIf([&](const F8Call& c) { return static_cast<bool>(c.Extents(rows, cols)); },
                [&] { return ScalesBytes(rows, cols); });
}

int seeml_hip_f8_quantize(const void* x, int dtype, uint64_t row_stride, uint64_t rows, uint64_t cols,
                          uint8_t* codes, uint8_t* scales, void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"F8Quantize"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Extents(rows, cols); !s) return s;
    if (!x || !codes || !scales) return call.Fail("null x, codes or scales");
    if (Status s = call.Stride("x", row_stride, rows, cols, dtype); !s) return s;
    if (Status s = call.Ranges({Rows("x", x, dtype, row_stride, rows, cols, false),
                                Codes("codes", codes, rows, cols, true), Scales("scales", scales, rows, cols, true)});
        !s)
      return s;
    if (Status s = call.OnDevice(x, stream, "x"); !s) return s;
    return F8Quantize(x, dtype, row_stride, rows, cols, codes, scales, On(stream));
  });
}

int seeml_hip_f8_quantize_weight(const void* w, int dtype, uint64_t row_stride, uint64_t rows, uint64_t cols,
                                 uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t,
                                 void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"F8QuantizeWeight"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Extents(rows, cols); !s) return s;
    if (!w) return call.Fail("null w");
    if (!codes != !scales || !codes_t != !scales_t) return call.Fail("codes and scales go together");
    if (!codes && !codes_t) return call.Fail("no output");
    if (Status s = call.Stride("w", row_stride, rows, cols, dtype); !s) return s;
    if (Status s = call.Ranges({Rows("w", w, dtype, row_stride, rows, cols, false),
                                Codes("codes", codes, rows, cols, true), Scales("scales", scales, rows, cols, true),
                                Codes("codes_t", codes_t, cols, rows, true),
                                Scales("scales_t", scales_t, cols, rows, true)});
        !s)
      return s;
    if (Status s = call.OnDevice(w, stream, "w"); !s) return s;
    return F8QuantizeWeight(w, dtype, row_stride, rows, cols, codes, scales, codes_t, scales_t, On(stream));
  });
}

int seeml_hip_f8_dequantize(const uint8_t* codes, const uint8_t* scales, void* x, int dtype, uint64_t row_stride,
                            uint64_t rows, uint64_t cols, void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"F8Dequantize"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Extents(rows, cols); !s) return s;
    if (!codes || !scales || !x) return call.Fail("null codes, scales or x");
    if (Status s = call.Stride("x", row_stride, rows, cols, dtype); !s) return s;
    if (Status s = call.Ranges({Codes("codes", codes, rows, cols), Scales("scales", scales, rows, cols),
                                Rows("x", x, dtype, row_stride, rows, cols, true)});
        !s)
      return s;
    if (Status s = call.OnDevice(codes, stream, "codes"); !s) return s;
    return F8Dequantize(codes, scales, x, dtype, row_stride, rows, cols, On(stream));
  });
}

uint64_t seeml_hip_gemm_f8_scratch(uint64_t M, uint64_t N, uint64_t K) {
  return SizeIf([&](const F8Call& c) { return c.Extents(M, N) && c.Extents(M, K) && c.Extents(N, K); },
                [&] { return GemmF8Scratch(M, N, K, 1); });
}

int seeml_hip_gemm_f8_nt(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                         const uint8_t* b_scales, void* C, int dtype, uint64_t c_stride, uint64_t M, uint64_t N,
                         uint64_t K, void* scratch, uint64_t scratch_bytes, void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"GemmF8"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Extents(M, K); !s) return s;
    if (Status s = call.Extents(N, K); !s) return s;
    if (Status s = call.Extents(M, N); !s) return s;
    if (!a_codes || !a_scales || !b_codes || !b_scales || !C) return call.Fail("null operand or C");
    if (Status s = call.Stride("C", c_stride, M, N, dtype); !s) return s;
    const uint64_t need = GemmF8Scratch(M, N, K, 1);
    if (Status s = call.Scratch(scratch, scratch_bytes, need); !s) return s;
    if (Status s = call.Ranges({Codes("a_codes", a_codes, M, K), Scales("a_scales", a_scales, M, K),
                                Codes("b_codes", b_codes, N, K), Scales("b_scales", b_scales, N, K),
                                Rows("C", C, dtype, c_stride, M, N, true),
                                {"scratch", need ? scratch : nullptr, need, true, 16}});
        !s)
      return s;
    if (Status s = call.OnDevice(a_codes, stream, "a_codes"); !s) return s;
    const GemmF8Args a{1, {a_codes, nullptr}, {a_scales, nullptr}, {b_codes, nullptr}, {b_scales, nullptr},
                       C, dtype, c_stride, M, N, K, scratch};
    return GemmF8(a, On(stream));
  });
}

uint64_t seeml_hip_gated_f8_scratch(uint64_t T, uint64_t D, uint64_t F) {
  return SizeIf([&](const F8Call& c) { return c.Extents(T, D) && c.Extents(T, F) && c.Extents(D, F); },
                [&] { return GatedF8Scratch(T, D, F); });
}

int seeml_hip_gated_f8_fwd(const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* wg_codes_t,
                           const uint8_t* wg_scales_t, const uint8_t* wu_codes_t, const uint8_t* wu_scales_t,
                           int act, void* h, int dtype, uint64_t h_stride, uint8_t* h_codes, uint8_t* h_scales,
                           uint8_t* g_codes, uint8_t* g_scales, uint8_t* u_codes, uint8_t* u_scales, uint64_t T,
                           uint64_t D, uint64_t F, void* scratch, uint64_t scratch_bytes, void* stream) {
  (void)scratch;
  (void)scratch_bytes;
  return Entry([&]() -> Status {
    const F8Call call{{"GatedF8Fwd"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Act(act); !s) return s;
    if (Status s = call.Extents(T, D); !s) return s;
    if (Status s = call.Extents(T, F); !s) return s;
    if (Status s = call.Extents(D, F); !s) return s;
    if (!x_codes || !x_scales || !wg_codes_t || !wg_scales_t || !wu_codes_t || !wu_scales_t)
      return call.Fail("null operand");
    if (!h_codes != !h_scales || !g_codes != !g_scales || !u_codes != !u_scales)
      return call.Fail("codes and scales go together");
    if (!h && !h_codes && !g_codes && !u_codes) return call.Fail("no output");
    if (h)
      if (Status s = call.Stride("h", h_stride, T, F, dtype); !s) return s;
    if (Status s = call.Ranges({Codes("x_codes", x_codes, T, D), Scales("x_scales", x_scales, T, D),
                                Codes("wg_codes_t", wg_codes_t, F, D), Scales("wg_scales_t", wg_scales_t, F, D),
                                Codes("wu_codes_t", wu_codes_t, F, D), Scales("wu_scales_t", wu_scales_t, F, D),
                                Rows("h", h, dtype, h ? h_stride : F, T, F, true),
                                Codes("h_codes", h_codes, T, F, true), Scales("h_scales", h_scales, T, F, true),
                                Codes("g_codes", g_codes, T, F, true), Scales("g_scales", g_scales, T, F, true),
                                Codes("u_codes", u_codes, T, F, true), Scales("u_scales", u_scales, T, F, true)});
        !s)
      return s;
    if (Status s = call.OnDevice(x_codes, stream, "x_codes"); !s) return s;
    return GatedF8Fwd({x_codes, x_scales, wg_codes_t, wg_scales_t, wu_codes_t, wu_scales_t, act, h, dtype, h_stride,
                       h_codes, h_scales, g_codes, g_scales, u_codes, u_scales, T, D, F},
                      On(stream));
  });
}

int seeml_hip_gated_f8_bwd(const void* dh, int dtype, uint64_t dh_stride, const uint8_t* g_codes,
                           const uint8_t* g_scales, const uint8_t* u_codes, const uint8_t* u_scales, int act,
                           const uint8_t* wg_codes, const uint8_t* wg_scales, const uint8_t* wu_codes,
                           const uint8_t* wu_scales, uint8_t* dg_codes, uint8_t* dg_scales, uint8_t* du_codes,
                           uint8_t* du_scales, void* h, uint64_t h_stride, void* dx, uint64_t dx_stride, uint64_t T,
                           uint64_t D, uint64_t F, void* scratch, uint64_t scratch_bytes, void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"GatedF8Bwd"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Act(act); !s) return s;
    if (Status s = call.Extents(T, D); !s) return s;
    if (Status s = call.Extents(T, F); !s) return s;
    if (Status s = call.Extents(D, F); !s) return s;
    if (!dh || !g_codes || !g_scales || !u_codes || !u_scales) return call.Fail("null dh, g or u");
    if (!dg_codes || !dg_scales || !du_codes || !du_scales) return call.Fail("null dg or du");
    if (dx && (!wg_codes || !wg_scales || !wu_codes || !wu_scales)) return call.Fail("dx without weights");
    if (Status s = call.Stride("dh", dh_stride, T, F, dtype); !s) return s;
    if (h)
      if (Status s = call.Stride("h", h_stride, T, F, dtype); !s) return s;
    if (dx)
      if (Status s = call.Stride("dx", dx_stride, T, D, dtype); !s) return s;
    const uint64_t need = dx ? GatedF8Scratch(T, D, F) : 0;
    if (Status s = call.Scratch(scratch, scratch_bytes, need); !s) return s;
    if (Status s = call.Ranges(
            {Rows("dh", dh, dtype, dh_stride, T, F, false), Codes("g_codes", g_codes, T, F),
             Scales("g_scales", g_scales, T, F), Codes("u_codes", u_codes, T, F), Scales("u_scales", u_scales, T, F),
             Codes("wg_codes", dx ? wg_codes : nullptr, D, F), Scales("wg_scales", dx ? wg_scales : nullptr, D, F),
             Codes("wu_codes", dx ? wu_codes : nullptr, D, F), Scales("wu_scales", dx ? wu_scales : nullptr, D, F),
             Codes("dg_codes", dg_codes, T, F, true), Scales("dg_scales", dg_scales, T, F, true),
             Codes("du_codes", du_codes, T, F, true), Scales("du_scales", du_scales, T, F, true),
             Rows("h", h, dtype, h ? h_stride : F, T, F, true), Rows("dx", dx, dtype, dx ? dx_stride : D, T, D, true),
             {"scratch", need ? scratch : nullptr, need, true, 16}});
        !s)
      return s;
    if (Status s = call.OnDevice(dh, stream, "dh"); !s) return s;
    const GatedF8BwdArgs a{dh, dtype, dh_stride, g_codes, g_scales, u_codes, u_scales, act, wg_codes, wg_scales,
                           wu_codes, wu_scales, dg_codes, dg_scales, du_codes, du_scales, h, h_stride, dx, dx_stride,
                           T, D, F, scratch};
    if (Status s = GatedF8BwdRows(a, On(stream)); !s || !dx) return s;
    // dx = [dg du] [Wg Wu]^T: one product over both pairs.
    const GemmF8Args p{2, {dg_codes, du_codes}, {dg_scales, du_scales}, {wg_codes, wu_codes}, {wg_scales, wu_scales},
                       dx, dtype, dx_stride, T, D, F, scratch};
    return GemmF8(p, On(stream));
  });
}

int seeml_hip_act_bwd_f8(const void* dy, int dtype, uint64_t dy_stride, const uint8_t* codes, const uint8_t* scales,
                         int act, void* dx, uint64_t dx_stride, uint64_t rows, uint64_t cols, void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"ActBwdF8"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Act(act); !s) return s;
    if (Status s = call.Extents(rows, cols); !s) return s;
    if (!dy || !codes || !scales || !dx) return call.Fail("null dy, codes, scales or dx");
    if (Status s = call.Stride("dy", dy_stride, rows, cols, dtype); !s) return s;
    if (Status s = call.Stride("dx", dx_stride, rows, cols, dtype); !s) return s;
    const Span in = Rows("dy", dy, dtype, dy_stride, rows, cols, false);
    const Span out = Rows("dx", dx, dtype, dx_stride, rows, cols, true);
    if (Status s = call.InPlace(in, dy_stride, out, dx_stride, rows); !s) return s;
    if (Status s = call.Ranges({in}); !s) return s;
    if (Status s = call.Ranges({out, Codes("codes", codes, rows, cols), Scales("scales", scales, rows, cols)}); !s)
      return s;
    if (Status s = call.OnDevice(dy, stream, "dy"); !s) return s;
    return ActBwdF8(dy, dtype, dy_stride, codes, scales, act, dx, dx_stride, rows, cols, On(stream));
  });
}

int seeml_hip_rms_norm_bwd_f8(const void* dy, int dtype, uint64_t dy_stride, const uint8_t* codes,
                              const uint8_t* scales, const float* gamma, const float* rstd, void* dx,
                              uint64_t dx_stride, uint64_t rows, uint64_t cols, void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"RmsNormBwdF8"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Extents(rows, cols); !s) return s;
    if (!dy || !codes || !scales || !gamma || !rstd || !dx)
      return call.Fail("null dy, codes, scales, gamma, rstd or dx");
    if (Status s = call.Stride("dy", dy_stride, rows, cols, dtype); !s) return s;
    if (Status s = call.Stride("dx", dx_stride, rows, cols, dtype); !s) return s;
    const Span in = Rows("dy", dy, dtype, dy_stride, rows, cols, false);
    const Span out = Rows("dx", dx, dtype, dx_stride, rows, cols, true);
    if (Status s = call.InPlace(in, dy_stride, out, dx_stride, rows); !s) return s;
    if (Status s = call.Ranges({in}); !s) return s;
    if (Status s = call.Ranges({out, Codes("codes", codes, rows, cols), Scales("scales", scales, rows, cols),
                                {"gamma", gamma, cols * 4, false, 4}, {"rstd", rstd, rows * 4, false, 4}});
        !s)
      return s;
    if (Status s = call.OnDevice(dy, stream, "dy"); !s) return s;
    return RmsNormBwdF8(dy, dtype, dy_stride, codes, scales, gamma, rstd, dx, dx_stride, rows, cols, On(stream));
  });
}

uint64_t seeml_hip_gemm_tn_f8_scratch(uint64_t T, uint64_t D, uint64_t r) {
  return SizeIf([&](const F8Call& c) { return c.Extents(T, D) && r >= 1 && r <= kMaxRank; },
                [&] { return GemmTnF8Scratch(T, D, r); });
}

int seeml_hip_gemm_tn_f8(const uint8_t* x_codes, const uint8_t* x_scales, const void* dt, int dtype,
                         uint64_t dt_stride, float* out, uint64_t T, uint64_t D, uint64_t r, void* scratch,
                         uint64_t scratch_bytes, void* stream) {
  return Entry([&]() -> Status {
    const F8Call call{{"GemmTnF8"}};
    if (Status s = call.Type(dtype); !s) return s;
    if (Status s = call.Extents(T, D); !s) return s;
    if (r == 0) return call.Fail("empty input");
    if (r > kMaxRank) return call.Fail("rank above " + std::to_string(kMaxRank));
    if (!x_codes || !x_scales || !dt || !out) return call.Fail("null x, dt or out");
    if (Status s = call.Stride("dt", dt_stride, T, r, dtype); !s) return s;
    const uint64_t need = GemmTnF8Scratch(T, D, r);
    if (Status s = call.Scratch(scratch, scratch_bytes, need); !s) return s;
    if (Status s = call.Ranges({Codes("x_codes", x_codes, T, D), Scales("x_scales", x_scales, T, D),
                                Rows("dt", dt, dtype, dt_stride, T, r, false), {"out", out, D * r * 4, true, 4},
                                {"scratch", need ? scratch : nullptr, need, true, 16}});
        !s)
      return s;
    if (Status s = call.OnDevice(x_codes, stream, "x_codes"); !s) return s;
    return GemmTnF8(x_codes, x_scales, dt, dtype, dt_stride, out, T, D, r, scratch, On(stream));
  });
}

}  // extern "C"
