// The 4-bit projections' entry points (kernel: proj_mx4_kernel.h).
//
//   y[m, n] = sum over blocks b of 32 of 2^(ex[m, b] + ew[n, b]) sum_i x[m, i] w[n, i]
//
// with x and w e2m1: what rounds is the fp32 sum and the one rounding to bf16.
// h3hip_proj_mx4 writes y token-major; h3hip_qkv_proj_mx4 treats it as Q | K | V heads and ends as
// h3hip_qkv_proj_i8 does: Q and K are h3hip_qk_norm_rope of h3hip_proj_mx4's result, bit for bit,
// or in H3HIP_ROUND_ONCE the norm and rotation of the fp32 sums. The linear forms take bf16 rows
// and round them on the way, one or two in the product's launch (few_mx4.hip), more in one before
// it.
#include "few_mx4.h"
#include "proj_mx4.h"

namespace h3hip {

namespace {

constexpr int kHeadDim = 128;
constexpr int kStepValues = 256;
constexpr int64_t kMaxStride = ((int64_t)1 << 31) / 256;

int64_t padded(int32_t in) { return ((int64_t)in + kStepValues - 1) / kStepValues * kStepValues; }

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

// What the bf16 rows and the weight of a linear call have to be.
int check_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* w_scale,
                 int32_t in) {
  const int64_t bytes = padded(in) / 2;
  H3_REQUIRE(x && w && w_scale, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(ldx >= in && ldw >= bytes && ldw % 16 == 0, H3HIP_EINVAL,
             "ldx %lld must cover a row, ldw %lld a row's bytes and be a multiple of 16",
             (long long)ldx, (long long)ldw);
  H3_REQUIRE(ldw < kMaxStride && bytes < kMaxStride, H3HIP_EINVAL,
             "256 rows of x or w exceed 2 GiB (in_features %d, ldw %lld)", in, (long long)ldw);
  H3_REQUIRE(aligned(x, 2) && aligned(w, 16) && aligned(w_scale, 4), H3HIP_EINVAL,
             "x must be 2-byte, w 16-byte and its scale 4-byte aligned");
  return H3HIP_OK;
}

int check_y(const void* y, int64_t ldy, int32_t out_features) {
  H3_REQUIRE(y != nullptr, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(ldy >= out_features && aligned(y, 2), H3HIP_EINVAL,
             "ldy %lld must cover a row, and y be 2-byte aligned", (long long)ldy);
  return H3HIP_OK;
}

// Geometry and tensors of a QKV call beside its operands.
bool heads_declined(int32_t head_dim, int32_t rot) {
  if (head_dim == kHeadDim && (rot == 96 || rot == 128)) return false;
  set_error("declined: head_dim %d / rot %d (needs head_dim 128, rot 96 or 128)", head_dim, rot);
  return true;
}
int check_heads(const void* q_gamma, const void* k_gamma, const void* rope_table, int32_t rounding,
                int32_t seq_len, int32_t seq_pad, int32_t heads, const void* q_out,
                const void* k_out, const void* v_out) {
  const bool plain = q_gamma == nullptr && k_gamma == nullptr;
  H3_REQUIRE(seq_len > 0 && heads > 0 && heads <= INT32_MAX / (3 * kHeadDim) &&
                 seq_pad >= seq_len && seq_pad % 128 == 0,
             H3HIP_EINVAL, "bad shape: seq_len %d seq_pad %d heads %d", seq_len, seq_pad, heads);
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
  return H3HIP_OK;
}

ProjArgs token_args(void* y, int64_t ldy, int32_t out_features, int32_t rows) {
  ProjArgs o{};
  o.q_out = static_cast<uint16_t*>(y);
  o.ldo = ldy;
  o.n_out = out_features;
  o.seq_len = rows;
  return o;
}

ProjArgs head_args(const void* q_gamma, const void* k_gamma, float eps, const void* rope_table,
                   int32_t rot, int32_t seq_len, int32_t seq_pad, int32_t heads, void* q_out,
                   void* k_out, void* v_out) {
  ProjArgs o{};
  o.q_gamma = static_cast<const uint16_t*>(q_gamma);
  o.k_gamma = static_cast<const uint16_t*>(k_gamma);
  o.table = rope_table;
  o.q_out = static_cast<uint16_t*>(q_out);
  o.k_out = static_cast<uint16_t*>(k_out);
  o.v_out = static_cast<uint16_t*>(v_out);
  o.eps = eps;
  o.rot = rot;
  o.seq_len = seq_len;
  o.seq_pad = seq_pad;
  o.heads = heads;
  return o;
}

// The product of two operands in 4 bits.
int product(const ProjArgs& o, const void* x, int64_t ldx, const void* x_scale, const void* w,
            int64_t ldw, const void* w_scale, int32_t in, int32_t n_total, int32_t rounding,
            bool plain, bool out, void* stream) {
  ProjMx4Args a{};
  a.out = o;
  a.x = static_cast<const uint8_t*>(x);
  a.w = static_cast<const uint8_t*>(w);
  a.x_scale = static_cast<const uint8_t*>(x_scale);
  a.w_scale = static_cast<const uint8_t*>(w_scale);
  a.ldx = ldx;
  a.ldw = ldw;
  a.in = in;
  a.n_total = n_total;
  return launch_proj_mx4_gemm(a, rounding, plain, out, as_stream(stream));
}

// Bytes of the codes of `rows` rows in a workspace; their scales follow.
int64_t code_bytes(int32_t rows, int32_t in) { return (int64_t)rows * (padded(in) / 2); }

// Whether an output lies on one of the few rows of x, which every workgroup of few_mx4_kernel
// reads while others store.
bool on_few_rows(const ProjArgs& o, const void* x, int64_t ldx, int32_t in, int32_t n_total, bool out) {
  auto meet = [](uintptr_t a, int64_t na, const void* b, int64_t nb) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(b);
    return a < at + (uintptr_t)nb && at < a + (uintptr_t)na;
  };
  for (int32_t r = 0; r < o.seq_len; r++) {
    const uintptr_t row = reinterpret_cast<uintptr_t>(x) + 2 * (uintptr_t)(r * ldx);
    if (out) {
      for (int32_t s = 0; s < o.seq_len; s++)
        if (meet(row, 2 * (int64_t)in, o.q_out + s * o.ldo, 2 * (int64_t)n_total)) return true;
    } else {
      const int64_t heads = 2 * (int64_t)o.heads * o.seq_pad * kHeadDim;
      for (const uint16_t* t : {o.q_out, o.k_out, o.v_out})
        if (meet(row, 2 * (int64_t)in, t, heads)) return true;
    }
  }
  return false;
}

// The product of bf16 rows: one or two rounded on the way, more into the workspace first.
int linear(const ProjArgs& o, const void* x, int64_t ldx, const void* w, int64_t ldw,
           const void* w_scale, int32_t in, int32_t n_total, int32_t rounding, bool plain, bool out,
           void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = h3hip_linear_mx4_workspace(o.seq_len, in);
  H3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
             H3HIP_EINVAL, "a workspace of %lld bytes, 16-byte aligned, is needed (%lld given)",
             (long long)need, (long long)(workspace ? workspace_bytes : 0));
  // Before the rows are rounded: what no tile shape takes, the largest does not.
  H3_REQUIRE(proj_mx4_fits(o.seq_len, n_total, kProjMx4Shapes[0]), H3HIP_EINVAL,
             "too many rows or channels for one launch (%d x %d)", o.seq_len, n_total);
  if (few_mx4_takes(o.seq_len, in)) {
    H3_REQUIRE(!on_few_rows(o, x, ldx, in, n_total, out), H3HIP_EINVAL,
               "an output overlaps x: of one or two rows the product reads x while it is written");
    FewMx4Args few{};
    few.x = static_cast<const uint16_t*>(x);
    few.w = static_cast<const uint8_t*>(w);
    few.w_scale = static_cast<const uint8_t*>(w_scale);
    few.q_out = o.q_out, few.k_out = o.k_out, few.v_out = o.v_out;
    few.ldx = ldx, few.ldw = ldw, few.ldy = o.ldo;
    few.rows = o.seq_len, few.cols = in, few.units = (int32_t)(padded(in) / 256);
    few.n_total = n_total, few.heads = o.heads, few.seq_pad = o.seq_pad;
    const int rc = launch_few_mx4(few, as_stream(stream));
    if (rc != H3HIP_OK || out) return rc;
    return launch_few_heads(o, rounding, plain, as_stream(stream));
  }
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scale = codes + code_bytes(o.seq_len, in);
  const int64_t ld = padded(in) / 2;
  const int rc = h3hip_quant_rows_mx4(x, ldx, o.seq_len, in, codes, ld, scale, stream);
  if (rc != H3HIP_OK) return rc;
  return product(o, codes, ld, scale, w, ldw, w_scale, (int32_t)padded(in), n_total, rounding, plain,
                 out, stream);
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
  int rc = check_operands(x, ldx, x_scale, w, ldw, w_scale, in_features);
  if (rc == H3HIP_OK) rc = check_y(y, ldy, out_features);
  if (rc != H3HIP_OK) return rc;
  return product(token_args(y, ldy, out_features, rows), x, ldx, x_scale, w, ldw, w_scale,
                 in_features, out_features, H3HIP_ROUND_REFERENCE, true, true, stream);
}

extern "C" int h3hip_qkv_proj_mx4(const void* x, int64_t ldx, const void* x_scale, const void* w,
                                  int64_t ldw, const void* w_scale, int32_t hidden,
                                  const void* q_gamma, const void* k_gamma, float eps,
                                  const void* rope_table, int32_t rot, int32_t rounding,
                                  int32_t seq_len, int32_t seq_pad, int32_t heads,
                                  int32_t head_dim, void* q_out, void* k_out, void* v_out,
                                  void* stream) {
  H3_REQUIRE(hidden > 0, H3HIP_EINVAL, "hidden must be positive (got %d)", hidden);
  if (heads_declined(head_dim, rot)) return H3HIP_DECLINED;
  if (hidden % kStepValues != 0) {
    set_error("declined: hidden %d (needs a multiple of 256; h3hip_quant_rows_mx4 pads rows with "
              "zeros)", hidden);
    return H3HIP_DECLINED;
  }
  int rc = check_heads(q_gamma, k_gamma, rope_table, rounding, seq_len, seq_pad, heads, q_out, k_out,
                       v_out);
  if (rc == H3HIP_OK) rc = check_operands(x, ldx, x_scale, w, ldw, w_scale, hidden);
  if (rc != H3HIP_OK) return rc;
  return product(head_args(q_gamma, k_gamma, eps, rope_table, rot, seq_len, seq_pad, heads, q_out,
                           k_out, v_out),
                 x, ldx, x_scale, w, ldw, w_scale, hidden, 3 * heads * kHeadDim, rounding,
                 !q_gamma && !k_gamma, false, stream);
}

extern "C" int64_t h3hip_linear_mx4_workspace(int32_t rows, int32_t in_features) {
  if (rows <= 0 || in_features <= 0 || few_mx4_takes(rows, in_features)) return 0;
  // What every call refuses (check_linear(), linear()).
  if (padded(in_features) / 2 >= kMaxStride || !proj_mx4_fits(rows, 1, kProjMx4Shapes[0])) return 0;
  const int64_t slabs = ((int64_t)in_features + 511) / 512, groups = ((int64_t)rows + 15) / 16;
  return code_bytes(rows, in_features) + 256 * slabs * groups;
}

extern "C" int h3hip_linear_mx4(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                const void* w_scale, int32_t in_features, int32_t out_features,
                                int32_t rows, void* y, int64_t ldy, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  H3_REQUIRE(in_features > 0 && out_features > 0 && rows >= 0, H3HIP_EINVAL,
             "bad shape: in_features %d out_features %d rows %d", in_features, out_features, rows);
  if (rows == 0) return H3HIP_OK;
  int rc = check_linear(x, ldx, w, ldw, w_scale, in_features);
  if (rc == H3HIP_OK) rc = check_y(y, ldy, out_features);
  if (rc != H3HIP_OK) return rc;
  return linear(token_args(y, ldy, out_features, rows), x, ldx, w, ldw, w_scale, in_features,
                out_features, H3HIP_ROUND_REFERENCE, true, true, workspace, workspace_bytes, stream);
}

extern "C" int h3hip_qkv_linear_mx4(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                    const void* w_scale, int32_t hidden, const void* q_gamma,
                                    const void* k_gamma, float eps, const void* rope_table,
                                    int32_t rot, int32_t rounding, int32_t seq_len, int32_t seq_pad,
                                    int32_t heads, int32_t head_dim, void* q_out, void* k_out,
                                    void* v_out, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  H3_REQUIRE(hidden > 0, H3HIP_EINVAL, "hidden must be positive (got %d)", hidden);
  if (heads_declined(head_dim, rot)) return H3HIP_DECLINED;
  int rc = check_heads(q_gamma, k_gamma, rope_table, rounding, seq_len, seq_pad, heads, q_out, k_out,
                       v_out);
  if (rc == H3HIP_OK) rc = check_linear(x, ldx, w, ldw, w_scale, hidden);
  if (rc != H3HIP_OK) return rc;
  return linear(head_args(q_gamma, k_gamma, eps, rope_table, rot, seq_len, seq_pad, heads, q_out,
                          k_out, v_out),
                x, ldx, w, ldw, w_scale, hidden, 3 * heads * kHeadDim, rounding,
                !q_gamma && !k_gamma, false, workspace, workspace_bytes, stream);
}
