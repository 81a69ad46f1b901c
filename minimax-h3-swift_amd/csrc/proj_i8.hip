// The int8 projections' entry points (kernel: proj_i8_kernel.h).
//
//   y[m, n] = ((sum_k x[m, k] w[n, k]) w_scale[n]) x_scale[m]
//
// with x and w int8 and the sum exact in int32 (in_features up to 131,071, whatever
// the values): what rounds is the sum's conversion to fp32, the two products with
// the scales and the one rounding to bf16. h3hip_proj_i8 writes y token-major;
// h3hip_qkv_proj_i8 treats it as Q | K | V heads and ends as h3hip_qkv_proj does, with
// the bf16 product normalised and rotated by the code of the bf16 path
// (proj_rows.h), so its Q and K are h3hip_qk_norm_rope of h3hip_proj_i8's result, bit
// for bit; in H3HIP_ROUND_ONCE the fp32 product is, and rounded at the store.
#include "proj_i8.h"

namespace h3hip {

namespace {

constexpr int kHeadDim = 128;
constexpr int kStepBytes = 128;
constexpr int kMaxIn = 131071;                      // x 128 x 128 stays below 2^31
constexpr int64_t kMaxStride = ((int64_t)1 << 31) / 256;

bool aligned(const void* p, uintptr_t to) {
  return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

// The reduction's checks shared by both entry points.
int check_operands(const void* x, int64_t ldx, const float* x_scale, const void* w, int64_t ldw,
                   const float* w_scale, int32_t in) {
  H3_REQUIRE(x && x_scale && w && w_scale, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(ldx >= in && ldx % 16 == 0 && ldw >= in && ldw % 16 == 0, H3HIP_EINVAL,
             "ldx %lld / ldw %lld must cover a row and be multiples of 16", (long long)ldx,
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

extern "C" int h3hip_proj_i8(const void* x, int64_t ldx, const float* x_scale, const void* w,
                             int64_t ldw, const float* w_scale, int32_t in_features,
                             int32_t out_features, int32_t rows, void* y, int64_t ldy,
                             void* stream) {
  H3_REQUIRE(in_features > 0 && out_features > 0 && rows >= 0, H3HIP_EINVAL,
             "bad shape: in_features %d out_features %d rows %d", in_features, out_features, rows);
  if (in_features % kStepBytes != 0 || in_features > kMaxIn) {
    set_error("declined: in_features %d (needs a multiple of 128, at most %d; h3hip_quant_rows "
              "pads rows with zeros)", in_features, kMaxIn);
    return H3HIP_DECLINED;
  }
  if (rows == 0) return H3HIP_OK;
  const int rc = check_operands(x, ldx, x_scale, w, ldw, w_scale, in_features);
  if (rc != H3HIP_OK) return rc;
  H3_REQUIRE(y != nullptr, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(ldy >= out_features && aligned(y, 2), H3HIP_EINVAL,
             "ldy %lld must cover a row, and y be 2-byte aligned", (long long)ldy);
  ProjI8Args a{};
  a.out.q_out = static_cast<uint16_t*>(y);
  a.out.ldo = ldy;
  a.out.n_out = out_features;
  a.out.seq_len = rows;
  a.x = static_cast<const int8_t*>(x);
  a.w = static_cast<const int8_t*>(w);
  a.x_scale = x_scale;
  a.w_scale = w_scale;
  a.ldx = ldx;
  a.ldw = ldw;
  a.in = in_features;
  a.n_total = out_features;
  return launch_proj_i8_gemm(a, H3HIP_ROUND_REFERENCE, true, true, as_stream(stream));
}

extern "C" int h3hip_qkv_proj_i8(const void* x, int64_t ldx, const float* x_scale, const void* w,
                                 int64_t ldw, const float* w_scale, int32_t hidden,
                                 const void* q_gamma, const void* k_gamma, float eps,
                                 const void* rope_table, int32_t rot, int32_t rounding,
                                 int32_t seq_len, int32_t seq_pad, int32_t heads,
                                 int32_t head_dim, void* q_out, void* k_out, void* v_out,
                                 void* stream) {
  H3_REQUIRE(hidden > 0, H3HIP_EINVAL, "hidden must be positive (got %d)", hidden);
  if (head_dim != kHeadDim || (rot != 96 && rot != 128) || hidden % kStepBytes != 0 ||
      hidden > kMaxIn) {
    set_error("declined: head_dim %d / rot %d / hidden %d (needs head_dim 128, rot 96 or 128, hidden "
              "a multiple of 128, at most %d; h3hip_quant_rows pads rows with zeros)",
              head_dim, rot, hidden, kMaxIn);
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
  ProjI8Args a{};
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
  a.x = static_cast<const int8_t*>(x);
  a.w = static_cast<const int8_t*>(w);
  a.x_scale = x_scale;
  a.w_scale = w_scale;
  a.ldx = ldx;
  a.ldw = ldw;
  a.in = hidden;
  a.n_total = 3 * heads * kHeadDim;
  return launch_proj_i8_gemm(a, rounding, plain, false, as_stream(stream));
}
