// The int8 projections' entry points, and the kernel for few rows.
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n]
//
// with x and w int8 and the sum exact in int32 (in_features up to 131,071, whatever
// the values): what rounds is the sum's conversion to fp32, the two products with
// the scales and the one rounding to bf16. h3hip_proj_i8 writes y token-major;
// h3hip_qkv_proj_i8 treats it as Q | K | V heads and ends as h3hip_qkv_proj does, with
// the bf16 product normalised and rotated by the code of the bf16 path
// (proj_rows.h), so its Q and K are h3hip_qk_norm_rope of h3hip_proj_i8's result, bit
// for bit.
//
// The kernel here is v_mfma_i32_16x16x64_i8 straight from global memory: W rows as
// the A operand, x rows as B, no LDS in the loop. A wave owns 16 channels and every
// kSplit-th 128-byte step of the reduction; the waves' partial sums meet in LDS. The
// order of k within a step is free as long as both operands share it: lane (g, lr)
// takes bytes 32 g .. 32 g + 31 of row lr for the step's two products, so that a row's
// 128-byte line is read by one instruction pair.
#include <climits>

#include "proj_i8.h"
#include "proj_rows.h"

namespace h3hip {

namespace {

constexpr int kHeadDim = 128;
constexpr int kStepBytes = 128;
constexpr int kRowTokens = 16;   // tokens of a workgroup
constexpr int64_t kMaxThreads = (int64_t)1 << 32;   // a launch has fewer

// kBlocks blocks of 16 channels a workgroup, kSplit waves for each.
template <int kBlocks, int kSplit>
struct FewRows {
  static constexpr int kWaves = kBlocks * kSplit, kThreads = 64 * kWaves;
  static constexpr int kChannels = 16 * kBlocks;
};

// This wave's part of the 16 x 16 product of W rows n0 .. and x rows m0 .., summed over
// the waves of the block into the first of them.
template <int kBlocks, int kSplit>
__device__ __forceinline__ i32x4 few_rows_sum(const ProjI8Args& a, int64_t n0, int64_t m0, int wave,
                                              int lane, i32x4 (*part)[64]) {
  const int block = wave % kBlocks, split = wave / kBlocks;
  const int lr = lane & 15, g = lane >> 4;
  // Rows past the last are the last one's: in bounds, and never stored.
  const int64_t n = min(n0 + 16 * block + lr, (int64_t)a.n_total - 1);
  const int64_t m = min(m0 + lr, (int64_t)a.out.seq_len - 1);
  const int8_t* wp = a.w + n * a.ldw + 32 * g;
  const int8_t* xp = a.x + m * a.ldx + 32 * g;
  i32x4 acc = {0, 0, 0, 0};
  for (int k = kStepBytes * split; k < a.in; k += kStepBytes * kSplit) {
    const i32x4 w0 = *reinterpret_cast<const i32x4*>(wp + k);
    const i32x4 w1 = *reinterpret_cast<const i32x4*>(wp + k + 16);
    const i32x4 x0 = *reinterpret_cast<const i32x4*>(xp + k);
    const i32x4 x1 = *reinterpret_cast<const i32x4*>(xp + k + 16);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, x0, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, x1, acc, 0, 0, 0);
  }
  if (kSplit > 1) {
    part[wave][lane] = acc;
    __syncthreads();
    if (split == 0) {
#pragma unroll
      for (int s = 1; s < kSplit; s++) acc += part[wave + kBlocks * s][lane];
    }
  }
  return acc;
}

// Sums of channels 4g .. +3 of a token, with their scales.
__device__ __forceinline__ f32x4 scaled(const i32x4& acc, float xs, const float (&ws)[4]) {
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] = (float)acc[i] * xs * ws[i];
  return y;
}

template <int kSplit>
__global__ __launch_bounds__(64 * kSplit) void proj_i8_rows_kernel(ProjI8Args a) {
  __shared__ i32x4 part[kSplit][64];
  const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tiles_n = (a.n_total + 15) / 16;
  const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * kRowTokens;
  const int64_t n0 = (int64_t)(blockIdx.x % tiles_n) * 16;
  const i32x4 acc = few_rows_sum<1, kSplit>(a, n0, m0, wave, lane, part);
  const int64_t m = m0 + lr, n = n0 + 4 * g;
  if (wave != 0 || m >= a.out.seq_len || n >= a.n_total) return;
  float ws[4];
#pragma unroll
  for (int i = 0; i < 4; i++) ws[i] = a.w_scale[min(n + i, (int64_t)a.n_total - 1)];
  const f32x4 y = scaled(acc, a.x_scale[m], ws);
  uint16_t* dst = a.out.q_out + m * a.out.ldo + n;
  const u32x2 v = {cvt_pk(y[0], y[1]), cvt_pk(y[2], y[3])};
  if (a.wide && n + 4 <= a.n_total) {
    *reinterpret_cast<u32x2*>(dst) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (n + i < a.n_total) dst[i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
  }
}

// One head and 16 tokens: eight blocks of 16 channels.
template <int kSplit, int kMode, int kHl, bool kPlain>
__global__ __launch_bounds__(512 * kSplit) void qkv_proj_i8_rows_kernel(ProjI8Args a) {
  constexpr int kBlocks = kHeadDim / 16;
  __shared__ i32x4 part[kBlocks * kSplit][64];
  __shared__ __attribute__((aligned(16))) uint16_t rows[kRowTokens * kHeadDim];
  constexpr int kRowWaves = kRowTokens / 8;
  __shared__ __attribute__((aligned(16))) RopeEntry tables[kRowWaves * 512];
  const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int heads3 = 3 * a.out.heads;
  const int m0 = (int)(blockIdx.x / heads3) * kRowTokens;
  const int n0 = (int)(blockIdx.x % heads3) * kHeadDim;
  if (m0 >= a.out.seq_len) {
    zero_tile_rows<kRowTokens, kHeadDim, 512 * kSplit>(a.out, threadIdx.x, m0, n0);
    return;
  }
  const i32x4 acc = few_rows_sum<kBlocks, kSplit>(a, n0, m0, wave, lane, part);
  if (wave < kBlocks) {
    const f32x4 w4 = *reinterpret_cast<const f32x4*>(a.w_scale + n0 + 16 * wave + 4 * g);
    const float ws[4] = {w4[0], w4[1], w4[2], w4[3]};
    const f32x4 y = scaled(acc, a.x_scale[min(m0 + lr, a.out.seq_len - 1)], ws);
    const int chunk = 2 * wave + (g >> 1);
    *reinterpret_cast<u32x2*>(rows + lr * kHeadDim + (chunk ^ e_swz(lr)) * 8 + 4 * (g & 1)) =
        u32x2{cvt_pk(y[0], y[1]), cvt_pk(y[2], y[3])};
  }
  __syncthreads();
  if (wave < kRowWaves)
    finish_tile_rows<kRowTokens, kHeadDim, kRowWaves, kMode, kHl, kPlain, false>(
        a.out, rows, tables, wave, lane, m0, n0);
}

template <int kSplit>
int launch_qkv_rows(const ProjI8Args& a, int32_t rounding, bool plain, hipStream_t st) {
  const int64_t tiles = (int64_t)(a.out.seq_pad / kRowTokens) * 3 * a.out.heads;
  H3_REQUIRE(tiles * 512 * kSplit < kMaxThreads, H3HIP_EINVAL,
             "too many rows x heads for one launch (%lld tiles)", (long long)tiles);
  const dim3 grid((unsigned)tiles), block(512 * kSplit);
  constexpr int kRef = H3HIP_ROUND_REFERENCE, kF32 = H3HIP_ROUND_FP32;
  if (plain)
    qkv_proj_i8_rows_kernel<kSplit, kRef, 8, true><<<grid, block, 0, st>>>(a);
  else if (rounding == kRef && a.out.rot == 128)
    qkv_proj_i8_rows_kernel<kSplit, kRef, 8, false><<<grid, block, 0, st>>>(a);
  else if (rounding == kRef)
    qkv_proj_i8_rows_kernel<kSplit, kRef, 6, false><<<grid, block, 0, st>>>(a);
  else if (a.out.rot == 128)
    qkv_proj_i8_rows_kernel<kSplit, kF32, 8, false><<<grid, block, 0, st>>>(a);
  else
    qkv_proj_i8_rows_kernel<kSplit, kF32, 6, false><<<grid, block, 0, st>>>(a);
  return check_launch("qkv_proj_i8_rows_kernel");
}

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
  H3_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(x_scale, 4) && aligned(w_scale, 16),
             H3HIP_EINVAL, "x, w and w_scale must be 16-byte aligned, x_scale 4-byte");
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
  a.wide = ldy % 8 == 0 && aligned(y, 16);
  const ProjI8Tile tile = pick_proj_i8_tile(rows, rows, out_features, false);
  if (tile != ProjI8Tile::kRows)
    return launch_proj_i8_gemm(a, tile, H3HIP_ROUND_REFERENCE, true, true, as_stream(stream));
  constexpr int kSplit = 8;
  const int64_t tiles = (((int64_t)rows + kRowTokens - 1) / kRowTokens) *
                        (((int64_t)out_features + 15) / 16);
  H3_REQUIRE(tiles * 64 * kSplit < kMaxThreads, H3HIP_EINVAL,
             "too many rows x channels for one launch (%d x %d)", rows, out_features);
  proj_i8_rows_kernel<kSplit><<<dim3((unsigned)tiles), 64 * kSplit, 0, as_stream(stream)>>>(a);
  return check_launch("proj_i8_rows_kernel");
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
  const int rc = check_operands(x, ldx, x_scale, w, ldw, w_scale, hidden);
  if (rc != H3HIP_OK) return rc;
  H3_REQUIRE(q_out && k_out && v_out, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(plain || (q_gamma && k_gamma && rope_table), H3HIP_EINVAL,
             "gammas and the rotation table must all be given (or both gammas NULL for the "
             "plain GEMM)");
  H3_REQUIRE(seq_len > 0 && heads > 0 && heads <= INT32_MAX / (3 * kHeadDim) &&
                 seq_pad >= seq_len && seq_pad % 128 == 0,
             H3HIP_EINVAL, "bad shape: seq_len %d seq_pad %d heads %d", seq_len, seq_pad, heads);
  H3_REQUIRE(rounding == H3HIP_ROUND_REFERENCE || rounding == H3HIP_ROUND_FP32, H3HIP_EINVAL,
             "unknown rounding mode %d", rounding);
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
  const ProjI8Tile tile = pick_proj_i8_tile(seq_len, seq_pad, a.n_total, true);
  if (tile != ProjI8Tile::kRows)
    return launch_proj_i8_gemm(a, tile, rounding, plain, false, as_stream(stream));
  return launch_qkv_rows<2>(a, rounding, plain, as_stream(stream));
}
