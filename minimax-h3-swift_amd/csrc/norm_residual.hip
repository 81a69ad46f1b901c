// The norms around a DiT block's attention, fused with its modulation, gate and residual.
//
//   before:  h = x rsqrt(mean x^2 + eps) gamma (1 + scale[s]) + shift[s]
//   after:   r = alpha x + gate[s] z,  z = y or y rsqrt(mean y^2 + eps) post_gamma,
//            and with a next norm h of r as above
//
// s is the row's segment (text, audio and video tokens are modulated apart). The norm is
// H3RMSNorm (Sources/H3Modules/Modulation.swift:116-120) over the hidden width. Everything is
// fp32 between the loads and the one rounding of r and of h; h is normalised from the fp32 r, not
// from the rounded one.
//
// Bound by HBM: before 4 bytes an element, after with a next norm 8 (31,885 x 5,120: 137 us, 4.8
// TB/s, and 264 us, 4.9; a copy of 1 GiB 5.1; 18,102 rows of 7,168 to 16,384 4.5-5.1 but for 4.2 of
// 9,000), of few rows by the launch (125 x 5,120: 3.8 us). So a
// row is read once and stays in registers through its sums, and the tables, which as rows are as long as x's, are held
// in registers too, by workers that take a range of consecutive rows each and reload the
// tables only where a segment begins. The next row's loads are in flight while one is summed (of
// widths up to 8,192).
// A worker is a workgroup of as many waves as the row has chunks of 512 elements (of 1,024 past
// 8,192): 8 elements a thread. That depends on the width alone, and sums add in one order, so a
// row's bits do not depend on the other rows of the call.
#include <climits>

#include "common.h"
#include "norm_rule.h"

namespace h3hip {

namespace {

constexpr int kMaxSegments = 16;
constexpr int kLaneElems = 8;              // consecutive elements of a thread in a chunk
constexpr int kMaxThreads = 1024;
constexpr int kMaxHidden = 2 * kMaxThreads * kLaneElems;

// What a launch needs where one segment holds every row: 120 bytes, because the host takes 0.9 us
// longer for a launch of 128 bytes of arguments and more (the kernel's use of the launch's
// dimensions counts 256 of them, so they are made of hidden here).
struct NormRows {
  const uint16_t* x;                       // r or h may be x or y
  const uint16_t* y;
  uint16_t* r;
  uint16_t* h;
  const uint16_t* __restrict__ gate;
  const uint16_t* __restrict__ post;
  const uint16_t* __restrict__ gamma;
  const uint16_t* __restrict__ scale;
  const uint16_t* __restrict__ shift;
  int64_t ldx, ldy, ldr, ldh;
  float alpha, eps;
  int32_t rows;
  uint16_t hidden, workers_cu;             // workgroups a CU
};
template <bool kMany>
struct NormArgs : NormRows {};
template <>
struct NormArgs<true> : NormRows {
  int64_t ld_gate, ld_scale, ld_shift;
  int32_t segments;
  int32_t starts[kMaxSegments];
};

// Waves of a row of `hidden` elements, and its workgroups (fewer where there are fewer rows).
template <int kChunks>
__host__ __device__ constexpr int waves_of(int hidden) {
  return (hidden + 64 * kLaneElems * kChunks - 1) / (64 * kLaneElems * kChunks);
}
__host__ __device__ constexpr int workers_of(int rows, int workers_cu) {
  const int most = kNormCus * workers_cu;
  return rows < most ? rows : most;
}

// 8 elements from k on, zeros past n. Rows may begin anywhere.
__device__ __forceinline__ u32x4 load8(const uint16_t* row, int k, int n) {
  if (k + 8 <= n) return *reinterpret_cast<const u32x4_any*>(row + k);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (k + i < n) v[i / 2] |= (uint32_t)row[k + i] << (16 * (i & 1));
  return v;
}

// kPast: past the caches, for what is not read again soon. r with a next norm's h beside it is: the
// next half reads h at once and r at its end (both and the rounding of h to 4 bits at 1,151 x 5,376
// 23.4 -> 22.2 us, 31,885 x 5,120 342 -> 339). h is not: stored past the caches it took 58 us
// instead of 87 alone (18,102 x 5,120 again and again) and 136 instead of 117 with its rounding.
template <bool kPast>
__device__ __forceinline__ void store8(uint16_t* row, int k, int n, u32x4 v) {
  if (k + 8 <= n) {
    if constexpr (kPast)
      __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(row + k));
    else
      *reinterpret_cast<u32x4_any*>(row + k) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (k + i < n) row[k + i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
}

__device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) f[2 * i] = bf16_lo(v[i]), f[2 * i + 1] = bf16_hi(v[i]);
}

__device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  return v;
}

// A uniform row number that the compiler makes no running addresses of: they took 8 registers a
// thread more, past the 80 that there are.
__device__ __forceinline__ int opaque(int row) {
  asm("" : "+s"(row));
  return row;
}

template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(
      (uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), kCtrl, 0xf, 0xf, true));
}

// The sum over a wave, in every lane: lanes of a row of 16 by shifts, then row 0 into 1 and 2
// into 3, then rows 0-1 into 2-3; the last lane holds all of it.
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp<0x111>(v);
  v += dpp<0x112>(v);
  v += dpp<0x114>(v);
  v += dpp<0x118>(v);
  v += dpp<0x142>(v);
  v += dpp<0x143>(v);
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

// kChunks chunks of a row a thread. kAfter: there is y; kPost: it is normalised; kNext: h is
// written (without kAfter always); kMany: rows of more than one segment.
template <int kChunks, bool kAfter, bool kPost, bool kNext, bool kMany>
__global__ __launch_bounds__(kMaxThreads)
__attribute__((amdgpu_waves_per_eu(norm_waves_simd(kChunks, kAfter, kPost, kNext, kMany))))
void norm_residual_kernel(NormArgs<kMany> a) {
  constexpr int kSums = (kPost ? 1 : 0) + (kNext ? 1 : 0);
  constexpr int kMaxWaves = kMaxThreads / 64;
  __shared__ __attribute__((aligned(16))) float part[2][kSums > 0 ? kSums : 1][kMaxWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int n = a.hidden, waves = waves_of<kChunks>(n);
  // Rows first to last - 1: as many for every worker, one more for the first of them. With the one
  // more spread evenly 18,102 x 5,120 takes 88 us before and 162 after with a next norm instead of 78 and
  // 152, 31,885 x 5,376 147 and 291 instead of 151 and 293: where in memory the workers stand.
  const uint32_t workers = (uint32_t)workers_of(a.rows, a.workers_cu), rows = (uint32_t)a.rows;
  const uint32_t share = rows / workers, more = rows - share * workers;
  const int first = (int)(blockIdx.x * share + min(blockIdx.x, more));
  const int last = first + (int)(share + (blockIdx.x < more ? 1 : 0));
  const int k0 = kLaneElems * (int)threadIdx.x;
  const int stride = 64 * kLaneElems * waves;
  const float inv_n = 1.0f / (float)n;
  // Slots of waves that do not exist add as zeros.
  if (waves > 1 && (int)threadIdx.x < 2 * (kSums > 0 ? kSums : 1) * kMaxWaves)
    (&part[0][0][0])[threadIdx.x] = 0.0f;
  if (waves > 1) __syncthreads();

  // The sum over the row; parity and which pick a slot that no thread still reads.
  auto row_sum = [&](float v, int parity, int which) __attribute__((always_inline)) {
    v = wave_sum(v);
    if (waves > 1) {
      if (lane == 0) part[parity][which][wave] = v;
      __syncthreads();
      const f32x4* p = reinterpret_cast<const f32x4*>(part[parity][which]);
      f32x4 t = p[0];
      for (int i = 1; 4 * i < waves; i++) t += p[i];
      v = (t[0] + t[1]) + (t[2] + t[3]);
    }
    return v;
  };

  u32x4 vx[kChunks], vy[kChunks];
  auto load_row = [&](int at, u32x4 (&tx)[kChunks], u32x4 (&ty)[kChunks]) __attribute__((always_inline)) {
    const int row = opaque(at);
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const int k = k0 + c * stride;
      tx[c] = load8(a.x + row * a.ldx, k, n);
      if constexpr (kAfter) ty[c] = load8(a.y + row * a.ldy, k, n);
    }
  };
  constexpr bool kAhead = kChunks == 1;    // two chunks a thread leave no registers for it
  if (kAhead) load_row(first, vx, vy);

  // gate and post gamma in one factor, gamma and 1 + scale in one, and the shift, of the
  // row's segment.
  float fg[kAfter ? kChunks : 1][8], fa[kNext ? kChunks : 1][8], fb[kNext ? kChunks : 1][8];
  auto load_tables = [&](int s) __attribute__((always_inline)) {
    int64_t gate_at = 0, scale_at = 0, shift_at = 0;
    if constexpr (kMany)
      gate_at = s * a.ld_gate, scale_at = s * a.ld_scale, shift_at = s * a.ld_shift;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const int k = k0 + c * stride;
      if constexpr (kAfter) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) fg[c][i] = 1.0f;
        if (a.gate) unpack(load8(a.gate + gate_at, k, n), fg[c]);
        if constexpr (kPost) {
          unpack(load8(a.post, k, n), t);
#pragma unroll
          for (int i = 0; i < 8; i++) fg[c][i] *= t[i];
        }
      }
      if constexpr (kNext) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) fa[c][i] = 1.0f, fb[c][i] = 0.0f;
        if (a.gamma) unpack(load8(a.gamma, k, n), fa[c]);
        if (a.scale) {
          unpack(load8(a.scale + scale_at, k, n), t);
#pragma unroll
          for (int i = 0; i < 8; i++) fa[c][i] *= 1.0f + t[i];
        }
        if (a.shift) unpack(load8(a.shift + shift_at, k, n), fb[c]);
      }
    }
  };
  int until = first;                       // the row at which the tables change
  // Of one segment; beside the next row's loads it would take two registers too many here.
  if (!kMany && !kAhead) load_tables(0);
  for (int row = first; row < last; row++) {
    if constexpr (!kMany) {
      if (kAhead && row == first) load_tables(0);
    } else {
      if (row >= until) {
        int s = 0;
        until = INT_MAX;
        for (int i = 1; i < a.segments; i++) {
          if (a.starts[i] <= row) s = i;
          else until = min(until, a.starts[i]);
        }
        load_tables(s);
      }
    }
    u32x4 nx[kChunks], ny[kChunks];
    if (!kAhead)
      load_row(row, vx, vy);
    else if (row + 1 < last)
      load_row(row + 1, nx, ny);
    const int parity = (row - first) & 1;

    float v[kChunks][8];                   // x, then r
#pragma unroll
    for (int c = 0; c < kChunks; c++) unpack(vx[c], v[c]);
    if constexpr (kAfter) {
      float rs = 1.0f;
      if constexpr (kPost) {
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
          float t[8];
          unpack(vy[c], t);
#pragma unroll
          for (int i = 0; i < 8; i++) sum += t[i] * t[i];
        }
        rs = rsqrtf(row_sum(sum, parity, 0) * inv_n + a.eps);
      }
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        float t[8];
        unpack(vy[c], t);
#pragma unroll
        for (int i = 0; i < 8; i++) v[c][i] = a.alpha * v[c][i] + fg[c][i] * (t[i] * rs);
        store8<kNext>(a.r + opaque(row) * a.ldr, k0 + c * stride, n, pack(v[c]));
      }
    }
    if constexpr (kNext) {
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) sum += v[c][i] * v[c][i];
      const float rs = rsqrtf(row_sum(sum, parity, kSums - 1) * inv_n + a.eps);
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = v[c][i] * rs * fa[c][i] + fb[c][i];
        store8<false>(a.h + opaque(row) * a.ldh, k0 + c * stride, n, pack(t));
      }
    }
    if constexpr (kAhead) {
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        vx[c] = nx[c];
        if constexpr (kAfter) vy[c] = ny[c];
      }
    }
  }
}

template <int kChunks, bool kAfter, bool kPost, bool kNext, bool kMany>
void launch_form(NormArgs<kMany>& a, hipStream_t st) {
  const int waves = waves_of<kChunks>(a.hidden);
  a.workers_cu = (uint16_t)norm_workers_cu(
      waves, a.rows, norm_waves_simd(kChunks, kAfter, kPost, kNext, kMany));
  const dim3 grid((unsigned)workers_of(a.rows, a.workers_cu));
  norm_residual_kernel<kChunks, kAfter, kPost, kNext, kMany><<<grid, 64 * waves, 0, st>>>(a);
}

template <int kChunks, bool kMany>
void launch_chunks(NormArgs<kMany>& a, hipStream_t st) {
  const bool next = a.h != nullptr;
  if (a.y == nullptr)
    launch_form<kChunks, false, false, true>(a, st);
  else if (a.post && next)
    launch_form<kChunks, true, true, true>(a, st);
  else if (a.post)
    launch_form<kChunks, true, true, false>(a, st);
  else if (next)
    launch_form<kChunks, true, false, true>(a, st);
  else
    launch_form<kChunks, true, false, false>(a, st);
}

template <bool kMany>
void launch(NormArgs<kMany>& a, hipStream_t st) {
  if (a.hidden <= kMaxThreads * kLaneElems) launch_chunks<1>(a, st);
  else launch_chunks<2>(a, st);
}

// Fills in the sizes and launches; a's tables are the first segment's.
int launch(NormArgs<true>& a, int32_t rows, int32_t hidden, float eps, const int32_t* starts,
           int32_t segments, void* stream) {
  a.rows = rows;
  a.hidden = (uint16_t)hidden;
  a.eps = eps;
  a.segments = segments;
  for (int i = 1; i < segments; i++) a.starts[i] = starts[i];
  // The last segment that begins at row 0, and whether another row's begins after it.
  int s = 0;
  while (s + 1 < segments && starts[s + 1] == 0) s++;
  if (s + 1 < segments && starts[s + 1] < rows) {
    launch<true>(a, as_stream(stream));
  } else {
    NormArgs<false> one{a};
    if (one.gate) one.gate += s * a.ld_gate;
    if (one.scale) one.scale += s * a.ld_scale;
    if (one.shift) one.shift += s * a.ld_shift;
    launch<false>(one, as_stream(stream));
  }
  return check_launch("norm_residual_kernel");
}

bool aligned2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

// A table's row stride; 0: every segment has the one row.
bool covers(int64_t ld, int32_t hidden) { return ld >= hidden || ld == 0; }

// Rows that an output overwrites have to be the same rows.
int check_in_place(const void* out, int64_t ldo, const void* in, int64_t ldi, int32_t rows) {
  H3_REQUIRE(out != in || ldo == ldi || rows == 1, H3HIP_EINVAL,
             "an output in place of an input needs its stride (%lld, not %lld)", (long long)ldi,
             (long long)ldo);
  return H3HIP_OK;
}

// Sizes and segments, which both entry points share.
int check_sizes(int32_t rows, int32_t hidden, const int32_t* starts, int32_t segments) {
  H3_REQUIRE(rows >= 0 && hidden > 0, H3HIP_EINVAL, "bad shape: rows %d hidden %d", rows, hidden);
  H3_REQUIRE(segments >= 1 && segments <= kMaxSegments, H3HIP_EINVAL,
             "segments %d must be 1 to %d", segments, kMaxSegments);
  H3_REQUIRE(starts != nullptr || segments == 1, H3HIP_EINVAL, "NULL segment starts");
  if (starts) {
    H3_REQUIRE(starts[0] == 0, H3HIP_EINVAL, "the first segment must start at row 0, not %d",
               starts[0]);
    for (int i = 1; i < segments; i++)
      H3_REQUIRE(starts[i] >= starts[i - 1], H3HIP_EINVAL,
                 "segment starts must not descend (%d after %d)", starts[i], starts[i - 1]);
  }
  if (hidden > kMaxHidden) {
    set_error("declined: hidden %d (at most %d)", hidden, kMaxHidden);
    return H3HIP_DECLINED;
  }
  return H3HIP_OK;
}

int check_norm(const h3hip_norm* norm, int32_t hidden, int32_t segments) {
  H3_REQUIRE(aligned2(norm->gamma) && aligned2(norm->scale) && aligned2(norm->shift), H3HIP_EINVAL,
             "tensors must be 2-byte aligned");
  H3_REQUIRE(segments == 1 || ((!norm->scale || covers(norm->ld_scale, hidden)) &&
                               (!norm->shift || covers(norm->ld_shift, hidden))),
             H3HIP_EINVAL, "ld_scale %lld and ld_shift %lld must cover a row or be 0",
             (long long)norm->ld_scale, (long long)norm->ld_shift);
  return H3HIP_OK;
}

void set_norm(NormArgs<true>& a, const h3hip_norm* norm) {
  a.gamma = static_cast<const uint16_t*>(norm->gamma);
  a.scale = static_cast<const uint16_t*>(norm->scale);
  a.shift = static_cast<const uint16_t*>(norm->shift);
  a.ld_scale = norm->ld_scale;
  a.ld_shift = norm->ld_shift;
}

}  // namespace

}  // namespace h3hip

using namespace h3hip;

extern "C" int h3hip_norm_modulate(const void* x, int64_t ldx, int32_t rows, int32_t hidden,
                                   const h3hip_norm* norm, float eps, const int32_t* starts,
                                   int32_t segments, void* h, int64_t ldh, void* stream) {
  int rc = check_sizes(rows, hidden, starts, segments);
  if (rc != H3HIP_OK) return rc;
  H3_REQUIRE(norm != nullptr, H3HIP_EINVAL, "NULL norm");
  rc = check_norm(norm, hidden, segments);
  if (rc != H3HIP_OK) return rc;
  H3_REQUIRE(ldx >= hidden && ldh >= hidden, H3HIP_EINVAL, "ldx %lld and ldh %lld must cover a row",
             (long long)ldx, (long long)ldh);
  if (rows == 0) return H3HIP_OK;
  H3_REQUIRE(x && h, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(aligned2(x) && aligned2(h), H3HIP_EINVAL, "tensors must be 2-byte aligned");
  rc = check_in_place(h, ldh, x, ldx, rows);
  if (rc != H3HIP_OK) return rc;
  NormArgs<true> a{};
  a.x = static_cast<const uint16_t*>(x);
  a.h = static_cast<uint16_t*>(h);
  a.ldx = ldx;
  a.ldh = ldh;
  set_norm(a, norm);
  return launch(a, rows, hidden, eps, starts, segments, stream);
}

extern "C" int h3hip_gated_residual(const void* x, int64_t ldx, const void* y, int64_t ldy,
                                    int32_t rows, int32_t hidden, const void* gate, int64_t ld_gate,
                                    const void* post_gamma, float residual_scale,
                                    const h3hip_norm* next, float eps, const int32_t* starts,
                                    int32_t segments, void* r, int64_t ldr, void* h, int64_t ldh,
                                    void* stream) {
  int rc = check_sizes(rows, hidden, starts, segments);
  if (rc != H3HIP_OK) return rc;
  if (next) {
    rc = check_norm(next, hidden, segments);
    if (rc != H3HIP_OK) return rc;
  }
  H3_REQUIRE(ldx >= hidden && ldy >= hidden && ldr >= hidden && (!next || ldh >= hidden) &&
                 (!gate || segments == 1 || covers(ld_gate, hidden)),
             H3HIP_EINVAL, "ldx %lld, ldy %lld, ldr %lld, ldh %lld and ld_gate %lld must cover a row",
             (long long)ldx, (long long)ldy, (long long)ldr, (long long)ldh, (long long)ld_gate);
  if (rows == 0) return H3HIP_OK;
  H3_REQUIRE(x && y && r && (!next || h), H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(aligned2(x) && aligned2(y) && aligned2(r) && aligned2(h) && aligned2(gate) &&
                 aligned2(post_gamma),
             H3HIP_EINVAL, "tensors must be 2-byte aligned");
  H3_REQUIRE(!next || r != h, H3HIP_EINVAL, "r and h must be two tensors");
  rc = check_in_place(r, ldr, x, ldx, rows);
  if (rc == H3HIP_OK) rc = check_in_place(r, ldr, y, ldy, rows);
  if (rc == H3HIP_OK && next) rc = check_in_place(h, ldh, x, ldx, rows);
  if (rc == H3HIP_OK && next) rc = check_in_place(h, ldh, y, ldy, rows);
  if (rc != H3HIP_OK) return rc;
  NormArgs<true> a{};
  a.x = static_cast<const uint16_t*>(x);
  a.y = static_cast<const uint16_t*>(y);
  a.r = static_cast<uint16_t*>(r);
  a.h = next ? static_cast<uint16_t*>(h) : nullptr;
  a.gate = static_cast<const uint16_t*>(gate);
  a.post = static_cast<const uint16_t*>(post_gamma);
  a.ldx = ldx;
  a.ldy = ldy;
  a.ldr = ldr;
  a.ldh = ldh;
  a.ld_gate = ld_gate;
  a.alpha = residual_scale;
  if (next) set_norm(a, next);
  return launch(a, rows, hidden, eps, starts, segments, stream);
}
