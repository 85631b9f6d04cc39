// Residual update and norms around a block, one pass over the rows:
//
//   hidden = residual_scale * residual + gate * branch'
//   normed = rms(hidden) * (offset + weight) * (1 + scale) + shift
//   branch' = branch, or rms(branch) * (offset + branch_weight)
//
// A row is read once, held in registers over its one or two sums of squares
// and written once: 4 M D elements move, which bounds every call of more than
// a few rows. 16384 rows of 4096 in bf16, all operands: 106 us, 5.1 TB/s (a copy
// of as much: 112); 4095 rows of 2049 in f16: 21 us, 3.2 TB/s (2048: 15 us, 4.4;
// an odd row starts at any address, and its last element takes a chunk more);
// one row of 4096: 3.4 us, 800 of 1024: 5.2, the latency of one pass. f32, 16384
// rows of 4096: 210 us, 5.1 TB/s. Longer rows than the registers take pass three
// times, an element a thread: 4000 rows of 20000 in bf16 380 us (16384: 102), of
// 16384 in f32 271; rows of fewer than 8 columns fill no thread: 100000 of 4, 0.4
// ms.
#include <climits>
#include <cmath>

#include "block.hpp"

namespace actune {
namespace {

struct NormArgs {
  actune_block_norm_args p;
  int64_t per_wg;  // rows of one workgroup (kernel of rows in registers)
  int64_t first;   // the launch's first row (kernel of rows of any length)
};

// Row of a modulation tensor that row m reads.
__device__ __forceinline__ int64_t mod_row(int64_t m, int64_t rows) {
  return rows ? (uint32_t)m / (uint32_t)rows : 0;  // (both below 2^31)
}

// Sum over the TPR threads of a row, in every thread. red: TPR / 64 floats.
// Two sums in a row take two buffers: then the one barrier inside is enough,
// since a thread that writes a buffer again has passed the barrier of the sum
// between, behind every read of the first.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if constexpr (TPR == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < TPR / 64; ++i) v += red[i];
  return v;
}

// TPR threads a row, CH chunks of 8 elements a thread: 8 TPR (CH - 1) < D <=
// 8 TPR CH, at least 8. The
// weights stay in registers over the rows of a workgroup, gate, scale and
// shift while the next row reads the same ones. Rounded only when stored: h goes
// into its norm as it was summed, in f32.
template <int DT, int TPR, int CH>
__global__ __launch_bounds__(TPR > 64 ? TPR : 256) void norm_rows(const NormArgs args) {
  constexpr int RPW = TPR > 64 ? 1 : 4;  // (waves of different rows must not share a barrier)
  constexpr int ES = DT == kF32 ? 4 : 2;
  __shared__ float red[2][TPR / 64];
  const actune_block_norm_args& p = args.p;
  const int D = (int)p.D, t = RPW > 1 ? (int)threadIdx.x % TPR : (int)threadIdx.x;
  int64_t m = (int64_t)blockIdx.x * args.per_wg + (RPW > 1 ? threadIdx.x / TPR : 0);
  const int64_t end = min((int64_t)(blockIdx.x + 1) * args.per_wg, p.M);
  const bool behind = p.branch && p.branch_weight;
  const float offset = p.weight_offset;

  // a row ends in its threads' last chunks: the end that a chunk sees, and the last one's place
  auto end_of = [&](int i, int at) { return i < CH - 1 ? at + 8 : D; };
  const int last = 8 * ((CH - 1) * TPR + t);

  Raw8<DT> w[CH], bw[CH], gate[CH], scale[CH], shift[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int at = 8 * (i * TPR + t), n = end_of(i, at);
    w[i] = bw[i] = gate[i] = scale[i] = shift[i] = zero_raw<DT>();
    if (at >= n) continue;
    if (p.weight) w[i] = near_raw<DT>(p.weight, at, n);
    if (behind) bw[i] = near_raw<DT>(p.branch_weight, at, n);
  }
  if (last > D - 8 && last < D) {
    end_raw<DT>(w[CH - 1], last, D);
    end_raw<DT>(bw[CH - 1], last, D);
  }
  int64_t g_at = -1, sc_at = -1, sh_at = -1;  // the modulation rows held
  int turn = 0;                               // the buffer of the next sum

  for (; m < end; m += RPW) {
    const void* res = byte_at(p.residual, m * p.residual_stride * ES);
    const void* br = byte_at(p.branch, m * p.branch_stride * ES);
    Raw8<DT> rr[CH], rb[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = 8 * (i * TPR + t), n = end_of(i, at);
      rr[i] = rb[i] = zero_raw<DT>();
      if (at >= n) continue;
      rr[i] = near_raw<DT>(res, at, n);
      if (p.branch) rb[i] = near_raw<DT>(br, at, n);
    }
    auto modulation = [&](const void* src, int64_t stride, int64_t rows, int64_t& held, Raw8<DT>(&to)[CH]) {
      if (!src) return;
      const int64_t r = mod_row(m, rows);
      if (r == held) return;
      held = r;
      const void* row = byte_at(src, r * stride * ES);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int at = 8 * (i * TPR + t), n = end_of(i, at);
        if (at < n) to[i] = near_raw<DT>(row, at, n);
      }
      if (last > D - 8 && last < D) end_raw<DT>(to[CH - 1], last, D);
    };
    if (p.branch) modulation(p.gate, p.gate_stride, p.gate_rows, g_at, gate);
    modulation(p.scale, p.scale_stride, p.scale_rows, sc_at, scale);
    modulation(p.shift, p.shift_stride, p.shift_rows, sh_at, shift);

    if (last > D - 8 && last < D) {
      end_raw<DT>(rr[CH - 1], last, D);
      end_raw<DT>(rb[CH - 1], last, D);
    }

    float r1 = 1.f;
    if (behind) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(raw_at<DT>(rb[i], j), raw_at<DT>(rb[i], j), s);
      s = row_sum<TPR>(s, red[turn]);
      turn ^= 1;
      r1 = 1.f / sqrtf(s / (float)D + p.eps);
    }
    float h[CH][8], s = 0.f;
    void* hid = p.hidden ? (void*)byte_at(p.hidden, m * D * ES) : nullptr;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = 8 * (i * TPR + t), n = end_of(i, at);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float y = raw_at<DT>(rb[i], j);
        if (behind) y = y * r1 * (offset + raw_at<DT>(bw[i], j));
        if (p.gate) y *= raw_at<DT>(gate[i], j);
        h[i][j] = p.branch ? fmaf(p.residual_scale, raw_at<DT>(rr[i], j), y) : p.residual_scale * raw_at<DT>(rr[i], j);
        s = fmaf(h[i][j], h[i][j], s);
      }
      if (hid && at < n) store_raw<DT>(hid, at, n, h[i]);
    }
    s = row_sum<TPR>(s, red[turn]);
    turn ^= 1;
    const float r2 = 1.f / sqrtf(s / (float)D + p.eps);
    void* out = (void*)byte_at(p.normed, m * D * ES);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = 8 * (i * TPR + t), end = end_of(i, at);
      if (at >= end) continue;
      float n[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n[j] = h[i][j] * r2;
        if (p.weight) n[j] *= offset + raw_at<DT>(w[i], j);
        if (p.scale) n[j] *= 1.f + raw_at<DT>(scale[i], j);
        if (p.shift) n[j] += raw_at<DT>(shift[i], j);
      }
      store_raw<DT>(out, at, end, n);
    }
  }
}

// Rows of any length, one workgroup each: three passes, the second and third
// over data that the caches hold.
constexpr int kLong = 1024;

template <int DT>
__global__ __launch_bounds__(kLong) void norm_long(const NormArgs args) {
  constexpr int ES = DT == kF32 ? 4 : 2;
  __shared__ float red[2][kLong / 64];
  const actune_block_norm_args& p = args.p;
  const int64_t D = p.D, m = args.first + blockIdx.x;
  const bool behind = p.branch && p.branch_weight;
  const void* res = byte_at(p.residual, m * p.residual_stride * ES);
  const void* br = byte_at(p.branch, m * p.branch_stride * ES);
  const void* gate = byte_at(p.gate, mod_row(m, p.gate_rows) * p.gate_stride * ES);
  const void* scale = byte_at(p.scale, mod_row(m, p.scale_rows) * p.scale_stride * ES);
  const void* shift = byte_at(p.shift, mod_row(m, p.shift_rows) * p.shift_stride * ES);
  float r1 = 1.f;
  if (behind) {
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < D; i += kLong) {
      const float y = load_as_f32<DT>(br, i);
      s = fmaf(y, y, s);
    }
    r1 = 1.f / sqrtf(row_sum<kLong>(s, red[0]) / (float)D + p.eps);
  }
  auto update = [&](int64_t i) {
    const float r = load_as_f32<DT>(res, i);
    if (!p.branch) return p.residual_scale * r;
    float y = load_as_f32<DT>(br, i);
    if (behind) y = y * r1 * (p.weight_offset + load_as_f32<DT>(p.branch_weight, i));
    if (p.gate) y *= load_as_f32<DT>(gate, i);
    return fmaf(p.residual_scale, r, y);
  };
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < D; i += kLong) {
    const float h = update(i);
    s = fmaf(h, h, s);
    if (p.hidden) store_out<DT>(p.hidden, m * D + i, h);
  }
  const float r2 = 1.f / sqrtf(row_sum<kLong>(s, red[1]) / (float)D + p.eps);
  for (int64_t i = threadIdx.x; i < D; i += kLong) {
    float n = update(i) * r2;
    if (p.weight) n *= p.weight_offset + load_as_f32<DT>(p.weight, i);
    if (p.scale) n *= 1.f + load_as_f32<DT>(scale, i);
    if (p.shift) n += load_as_f32<DT>(shift, i);
    store_out<DT>(p.normed, m * D + i, n);
  }
}

// (a dispatch holds less than 2^32 threads: rows of few columns can be more)
template <int DT>
void launch_long(NormArgs a, hipStream_t st) {
  for (const int64_t most = 1 << 21; a.first < a.p.M; a.first += most) {
    const int64_t rows = a.p.M - a.first;
    norm_long<DT><<<dim3((unsigned)(rows < most ? rows : most)), kLong, 0, st>>>(a);
  }
}

template <int DT, int TPR, int CH>
void launch_rows(NormArgs a, hipStream_t st) {
  constexpr int RPW = TPR > 64 ? 1 : 4;
  const int64_t wgs = (a.p.M + RPW - 1) / RPW, most = 8 * kCus;
  const int64_t turns = (wgs + most - 1) / most;
  a.per_wg = turns * RPW;
  const int64_t grid = (a.p.M + a.per_wg - 1) / a.per_wg;
  norm_rows<DT, TPR, CH><<<dim3((unsigned)grid), TPR > 64 ? TPR : 256, 0, st>>>(a);
}

// Threads of a row by its length. One chunk a thread is the lowest latency while
// rows are short (1024: 4.0 us for 64 rows with 128 threads, 4.4 with 64 and two
// chunks, the same 44 for 32768); two chunks a thread and fewer threads at each
// barrier carry more rows at once above (4096: 4.5 us against 4.4 for one row
// with 512 threads, 9.1 against 10.5 for 1000, 112 against 114 for 16384; 2049:
// 21 against 28 for 4095; 8192: 5.6 against 6.0 for 100 with 1024, 105 against
// 133 for 8192). Two chunks of f32 in 1024 threads do not fit the registers.
template <int DT>
void launch_norm(const actune_block_norm_args& p, hipStream_t st) {
  const NormArgs a{p, 0, 0};
  const int64_t D = p.D;
  if (D < 8) launch_long<DT>(a, st);  // (a row in registers is eights)
  else if (D <= 512) launch_rows<DT, 64, 1>(a, st);
  else if (D <= 1024) launch_rows<DT, 128, 1>(a, st);
  else if (D <= 2048) launch_rows<DT, 256, 1>(a, st);
  else if (D <= 4096) launch_rows<DT, 256, 2>(a, st);
  else if (D <= 8192) launch_rows<DT, 512, 2>(a, st);
  else if (D <= 16384 && DT != kF32) launch_rows<DT, DT != kF32 ? 1024 : 512, 2>(a, st);
  else launch_long<DT>(a, st);
}

}  // namespace
}  // namespace actune

using namespace actune;

extern "C" int actune_block_norm(const actune_block_norm_args* args, void* stream) {
  block_clear_error();
  if (!args) return block_fail("null pointer");
  const actune_block_norm_args& p = *args;
  if (p.dtype != kBF16 && p.dtype != kF16 && p.dtype != kF32) return block_fail("unsupported dtype");
  if (p.M < 0 || p.M > INT_MAX || p.D <= 0 || p.D > INT_MAX) return block_fail("invalid dimensions");
  const int64_t most = INT64_MAX / 16 / (p.M + 1);
  for (int64_t s : {p.residual_stride, p.branch_stride, p.gate_stride, p.scale_stride, p.shift_stride})
    if (s < 0 || s > most) return block_fail("invalid row stride");
  for (int64_t r : {p.gate_rows, p.scale_rows, p.shift_rows})
    if (r < 0 || r > INT_MAX) return block_fail("invalid rows of a modulation row");
  if (!(p.eps >= 0.f) || !std::isfinite(p.eps)) return block_fail("eps must be finite and not negative");
  if (!std::isfinite(p.residual_scale) || !std::isfinite(p.weight_offset)) return block_fail("scales must be finite");
  if (!p.branch && (p.branch_weight || p.gate)) return block_fail("gate and branch_weight need a branch");
  if (p.M == 0) return kOk;
  if (!p.residual || !p.normed) return block_fail("null pointer");
  const uintptr_t es = p.dtype == kF32 ? 4 : 2;
  for (const void* t : {p.residual, p.branch, p.branch_weight, p.weight, p.gate, p.scale, p.shift,
                        (const void*)p.hidden, (const void*)p.normed})
    if (!is_aligned(t, es)) return block_fail("misaligned operand");
  hipStream_t st = (hipStream_t)stream;
  if (p.dtype == kBF16) launch_norm<kBF16>(p, st);
  else if (p.dtype == kF16) launch_norm<kF16>(p, st);
  else launch_norm<kF32>(p, st);
  return block_status();
}
