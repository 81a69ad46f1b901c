// The 4-bit projections' entry points (kernel: proj_mx4_kernel.h).
//
//   y[m, n] = sum over blocks b of 32 of 2^(ex[m, b] + ew[n, b]) sum_i x[m, i] w[n, i]
//
// with x and w e2m1: what rounds is the fp32 sum and the one rounding to bf16.
// h3hip_proj_mx4 writes y token-major; h3hip_qkv_proj_mx4 treats it as Q | K | V heads and ends as
// h3hip_qkv_proj_i8 does: Q and K are h3hip_qk_norm_rope of h3hip_proj_mx4's result, bit for bit,
// or in H3HIP_ROUND_ONCE the norm and rotation of the fp32 sums.
#include "proj_mx4.h"

namespace h3hip {

namespace {

constexpr int kHeadDim = 128;
constexpr int kStepValues = 256;
constexpr int64_t kMaxStride = ((int64_t)1 << 31) / 256;

bool aligned(const void* p, uintptr_t to) {
  return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

// The reduction's checks shared by both entry points.
int check_operands(const void* x, int64_t ldx, const void* x_scale, const void* w, int64_t ldw,
                   const void* w_scale, int32_t in) {
  H3_REQUIRE(x && x_scale && w && w_scale, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(ldx >= in / 2 && ldx % 16 == 0 && ldw >= in / 2 && ldw % 16 == 0, H3HIP_EINVAL,
             "ldx %lld / ldw %lld must cover a row's bytes and be multiples of 16", (long long)ldx,
             (long long)ldw);
  // A tile's rows are reached with 32-bit offsets from its first.
  H3_REQUIRE(ldx < kMaxStride && ldw < kMaxStride, H3HIP_EINVAL,
             "256 rows of x or w exceed 2 GiB (ldx %lld, ldw %lld)", (long long)ldx, (long long)ldw);
  H3_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(x_scale, 4) && aligned(w_scale, 4),
             H3HIP_EINVAL, "x and w must be 16-byte aligned, their scales 4-byte");
  return H3HIP_OK;
}

}  // namespace

}  // namespace h3hip

using namespace h3hip;

extern "C" int h3hip_proj_mx4(const void* x, int64_t ldx, const void* x_scale, const void* w,
                              int64_t ldw, const void* w_scale, int32_t in_features,
                              int32_t out_features, int32_t rows, void* y, int64_t ldy,
                              void* stream) {
  H3_REQUIRE(in_features > 0 && out_features > 0 && rows >= 0, H3HIP_EINVAL,
             "bad shape: in_features %d out_features %d rows %d", in_features, out_features, rows);
  if (in_features % kStepValues != 0) {
    set_error("declined: in_features %d (needs a multiple of 256; h3hip_quant_rows_mx4 pads rows "
              "with zeros)", in_features);
    return H3HIP_DECLINED;
  }
  if (rows == 0) return H3HIP_OK;
  const int rc = check_operands(x, ldx, x_scale, w, ldw, w_scale, in_features);
  if (rc != H3HIP_OK) return rc;
  H3_REQUIRE(y != nullptr, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(ldy >= out_features && aligned(y, 2), H3HIP_EINVAL,
             "ldy %lld must cover a row, and y be 2-byte aligned", (long long)ldy);
  ProjMx4Args a{};
  a.out.q_out = static_cast<uint16_t*>(y);
  a.out.ldo = ldy;
  a.out.n_out = out_features;
  a.out.seq_len = rows;
  a.x = static_cast<const uint8_t*>(x);
  a.w = static_cast<const uint8_t*>(w);
  a.x_scale = static_cast<const uint8_t*>(x_scale);
  a.w_scale = static_cast<const uint8_t*>(w_scale);
  a.ldx = ldx;
  a.ldw = ldw;
  a.in = in_features;
  a.n_total = out_features;
  return launch_proj_mx4_gemm(a, H3HIP_ROUND_REFERENCE, true, true, as_stream(stream));
}

extern "C" int h3hip_qkv_proj_mx4(const void* x, int64_t ldx, const void* x_scale, const void* w,
                                  int64_t ldw, const void* w_scale, int32_t hidden,
                                  const void* q_gamma, const void* k_gamma, float eps,
                                  const void* rope_table, int32_t rot, int32_t rounding,
                                  int32_t seq_len, int32_t seq_pad, int32_t heads,
                                  int32_t head_dim, void* q_out, void* k_out, void* v_out,
                                  void* stream) {
  H3_REQUIRE(hidden > 0, H3HIP_EINVAL, "hidden must be positive (got %d)", hidden);
  if (head_dim != kHeadDim || (rot != 96 && rot != 128) || hidden % kStepValues != 0) {
    set_error("declined: head_dim %d / rot %d / hidden %d (needs head_dim 128, rot 96 or 128, hidden "
              "a multiple of 256; h3hip_quant_rows_mx4 pads rows with zeros)", head_dim, rot, hidden);
    return H3HIP_DECLINED;
  }
  const bool plain = q_gamma == nullptr && k_gamma == nullptr;
  H3_REQUIRE(seq_len > 0 && heads > 0 && heads <= INT32_MAX / (3 * kHeadDim) &&
                 seq_pad >= seq_len && seq_pad % 128 == 0,
             H3HIP_EINVAL, "bad shape: seq_len %d seq_pad %d heads %d", seq_len, seq_pad, heads);
  const int rc = check_operands(x, ldx, x_scale, w, ldw, w_scale, hidden);
  if (rc != H3HIP_OK) return rc;
  H3_REQUIRE(q_out && k_out && v_out, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(plain || (q_gamma && k_gamma && rope_table), H3HIP_EINVAL,
             "gammas and the rotation table must all be given (or both gammas NULL for the "
             "plain GEMM)");
  H3_REQUIRE(rounding == H3HIP_ROUND_REFERENCE || rounding == H3HIP_ROUND_FP32 ||
                 rounding == H3HIP_ROUND_ONCE,
             H3HIP_EINVAL, "unknown rounding mode %d", rounding);
  H3_REQUIRE(aligned(q_out, 16) && aligned(k_out, 16) && aligned(v_out, 16) &&
                 (plain || (aligned(rope_table, 16) && aligned(q_gamma, 16) && aligned(k_gamma, 16))),
             H3HIP_EINVAL, "tensors must be 16-byte aligned");
  ProjMx4Args a{};
  a.out.q_gamma = static_cast<const uint16_t*>(q_gamma);
  a.out.k_gamma = static_cast<const uint16_t*>(k_gamma);
  a.out.table = rope_table;
  a.out.q_out = static_cast<uint16_t*>(q_out);
  a.out.k_out = static_cast<uint16_t*>(k_out);
  a.out.v_out = static_cast<uint16_t*>(v_out);
  a.out.eps = eps;
  a.out.rot = rot;
  a.out.seq_len = seq_len;
  a.out.seq_pad = seq_pad;
  a.out.heads = heads;
  a.x = static_cast<const uint8_t*>(x);
  a.w = static_cast<const uint8_t*>(w);
  a.x_scale = static_cast<const uint8_t*>(x_scale);
  a.w_scale = static_cast<const uint8_t*>(w_scale);
  a.ldx = ldx;
  a.ldw = ldw;
  a.in = hidden;
  a.n_total = 3 * heads * kHeadDim;
  return launch_proj_mx4_gemm(a, rounding, plain, false, as_stream(stream));
}
