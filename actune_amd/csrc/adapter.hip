// Low-rank adapters of many requests beside a shared projection:
//
//   out[m] = y[m] + scaling[id] * B[id] (A[id] x[m]),  id = ids[m / ids_rows]
//
// Two launches (or one for few tokens with small adapters, adapter_one). down:
// low[m] = A[id] x[m] in f32, K split over workgroups, each split's sums to the
// workspace. up: adds the splits, and out = y + scaling * B low.
//
// Both are matrix products over tiles of 16 tokens. A workgroup takes NT of
// them (or a single token where tokens are few) and goes over the distinct ids
// of its tokens; an adapter's matrix is read straight from memory, 16 bytes a
// lane, as the MFMA's operand, once for all its tiles with a token of that id,
// and the columns of the tokens that name it are kept. Tokens of one request
// stand side by side, so that a workgroup meets one or two ids where requests
// have tens of tokens; it goes through more of them one after the other. Rows of
// different ids never meet in a sum: one adapter's infinities stay with its
// requests.
//
// Bound by x, y and out: the adapters are re-read from L2 once for 64 tokens,
// and the next step's operands are requested before this one's products. 8192
// tokens of 8 requests, 4096 to 11008 columns, rank 64: 26 us down (67 MB of x,
// 2.5 TB/s: its wait is for the operands of A beside them, 35 us with 32 tokens
// a workgroup) and 98 us up (361 MB of y and out, 3.7 TB/s; a copy of as much
// takes 75). 12 tokens with an adapter each, 4096 to 4096, rank 16: one launch of
// 7.4 us. Single tokens with an adapter each are slow above 64, where a workgroup
// has 16 of them: 64, 65, 128 and 256 of them, same sizes, take 10, 35, 49 and 51
// us a call.
#include <climits>

#include "block.hpp"

namespace actune {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxRank = 128;
// token tiles of a workgroup with many tokens, by product: what their operands leave registers for
constexpr int kDownTiles = 4;
constexpr int up_tiles(int64_t R) { return R > 64 ? 2 : 4; }

struct AdapterArgs {
  actune_adapter_args p;
  float* part;       // [splits][M][RP] f32
  int RP;            // rank in whole tiles of 16
  int splits;        // K splits of the first product
  int chunk;         // K elements of one split
  int down_tokens;   // of a workgroup
  int up_tokens;
  int columns;       // of a workgroup of the second product
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Workgroup (x, y) of a grid whose consecutive items (y fastest) stay on an
// XCD, so that the tokens of a request find its adapter in one L2 (up: 99 us ->
// 97 and 9.5 -> 8.6 with 408 tokens; down is not helped, 30 -> 32).
__device__ __forceinline__ int2 item() {
  const int n = (int)(gridDim.x * gridDim.y), id = (int)(blockIdx.x + gridDim.x * blockIdx.y);
  const int x = id % kXcdCount, rest = n % kXcdCount, o = x * (n / kXcdCount) + min(x, rest) + id / kXcdCount;
  return make_int2((int)((uint32_t)o / gridDim.y), (int)((uint32_t)o % gridDim.y));
}

template <int DT>
__device__ __forceinline__ f32x4 mfma16(u16x8 a, u16x8 b, f32x4 c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Calls f(id, tokens) once for each distinct id in [0, L) among the wave's
// lanes, with the lanes (tokens of the workgroup) that hold it as bits.
template <typename F>
__device__ __forceinline__ void each_id(int id, int L, F f) {
  uint64_t left = __ballot(id >= 0 && id < L);
  while (left) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t same = __ballot(id == cur);
    left &= ~same;
    f(cur, same);
  }
}
// The id of the workgroup's token `lane`, -1 past its tokens.
__device__ __forceinline__ int token_id(const actune_adapter_args& p, int tokens, int64_t m0, int lane) {
  const int64_t m = m0 + lane;  // (below 2^31)
  return lane < tokens && m < p.M ? p.ids[(uint32_t)m / (uint32_t)p.ids_rows] : -1;
}
// two values to the 16-bit type, toward zero, a in the low half
template <int DT>
__device__ __forceinline__ uint32_t toward_zero(float a, float b) {
  if constexpr (DT == kBF16) return (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xffff0000u);
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
__device__ __forceinline__ u16x8 load8(const uint16_t* p) { return *(const u16x8_any*)p; }

// down: one split of K, the four waves a quarter each in steps of 64 (two MFMAs
// a step, of 32: the four lanes of a row read 64 consecutive bytes). RT: 16-row tiles of the rank at a time.
template <int DT, int RT, int NT>
__global__ __launch_bounds__(64 * kWaves) void adapter_down(const AdapterArgs args) {
  const actune_adapter_args& p = args.p;
  constexpr int TOK = 16 * NT;
  __shared__ float sums[kWaves][16 * RT][TOK + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, q = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * args.down_tokens;
  const int K = (int)p.K, R = (int)p.R, L = (int)p.L;
  const int k0 = (int)blockIdx.y * args.chunk, k1 = min(K, k0 + args.chunk);
  const int id = token_id(p, args.down_tokens, m0, lane);
  // rows past the workgroup's tokens read its first one's: their columns are not kept
  const uint16_t* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = 16 * t + col;
    x[t] = (const uint16_t*)p.x + (c < args.down_tokens && m0 + c < p.M ? m0 + c : m0) * p.x_stride;
  }
  for (int r0 = 0; r0 < args.RP; r0 += 16 * RT) {
    for (int e = threadIdx.x; e < kWaves * 16 * RT * (TOK + 1); e += 64 * kWaves) (&sums[0][0][0])[e] = 0.f;
    __syncthreads();
    each_id(id, L, [&](int cur, uint64_t same) {
      f32x4 acc[NT][RT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      const uint16_t* a[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = r0 + 16 * i + col;
        a[i] = (const uint16_t*)p.a + ((int64_t)cur * R + (r < R ? r : 0)) * K;  // (rows past the rank are not kept)
      }
      u16x8 av[2][RT], xv[2][NT];
      // operands of columns k + 8 q .. + 7 and 32 on, all tiles' (a branch around
      // those without this id would make each wait one for every load)
      auto fetch = [&](int k) {
        const int at = k + 8 * q;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int t = 0; t < NT; ++t) xv[h][t] = load8(x[t] + at + 32 * h);
#pragma unroll
          for (int i = 0; i < RT; ++i) av[h][i] = load8(a[i] + at + 32 * h);
        }
      };
      auto multiply = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[t][i] = mfma16<DT>(av[h][i], xv[h][t], acc[t][i]);
      };
      int k = k0 + 64 * wave;
      const int whole = k1 - 63;  // a step from below here is whole
      if (k < whole) fetch(k);
      for (; k + 64 * kWaves < whole; k += 64 * kWaves) {
        multiply();
        fetch(k + 64 * kWaves);
      }
      if (k < whole) {
        multiply();
        k += 64 * kWaves;
      }
      if (k < k1) {  // zeros past K's end
        const int at = k + 8 * q;
        const u16x8 none = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool any = at + 32 * h < k1;
#pragma unroll
          for (int i = 0; i < RT; ++i) av[h][i] = any ? load_raw<DT>(a[i], at + 32 * h, k1).v : none;
#pragma unroll
          for (int t = 0; t < NT; ++t) xv[h][t] = any ? load_raw<DT>(x[t], at + 32 * h, k1).v : none;
        }
        multiply();
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if ((same >> (16 * t + col)) & 1)
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wave][16 * i + 4 * q + e][16 * t + col] = acc[t][i][e];
    });
    __syncthreads();
    for (int e = threadIdx.x; e < args.down_tokens * 16 * RT; e += 64 * kWaves) {
      const int c = e / (16 * RT), r = e % (16 * RT);
      if (m0 + c >= p.M || r0 + r >= args.RP) continue;
      float s = sums[0][r][c];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) s += sums[w][r][c];
      args.part[((int64_t)blockIdx.y * p.M + m0 + c) * args.RP + r0 + r] = r0 + r < R ? s : 0.f;
    }
    __syncthreads();
  }
}

// up: a wave takes 64 columns at a time: four products t whose rows stand for
// columns 32 (t / 2) + 8 (row / 4) + 4 (t % 2) + row % 4, so that a lane ends
// with two runs of 8 columns of its token, and the four lanes of a token with 64
// consecutive bytes of each half. low is held as hi + lo of the 16-bit type under
// a power of two that brings its row's largest finite value to the type's middle
// (f16: below its end by the factor that keeps small values out of its
// subnormals; bf16: where 128 products of its largest values stay finite): no
// range is lost, and the second product's error stays near f32's (2^-16 of a
// value in bf16, 2^-21 in f16). hi is rounded toward zero, lo has its sign, and
// neither is zero where low is not: an infinity of B then gives both products
// the formula's sign, where a zero or another sign would make their sum NaN.
template <int DT, int KS, int NT>
__global__ __launch_bounds__(64 * kWaves) void adapter_up(const AdapterArgs args) {
  const actune_adapter_args& p = args.p;
  constexpr int TOK = 16 * NT, CH = 4 * KS;  // tokens; 8-element chunks of a row of low
  __shared__ u16x8 low[NT][KS][2][64];       // operand fragments of hi and lo
  __shared__ float2 by[TOK];                 // a token's scaling, and the power of two that its low is short of
  constexpr int kTop = DT == kF16 ? 14 : -9;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, q = lane >> 4;
  const int2 wg = item();
  const int64_t m0 = (int64_t)wg.x * args.up_tokens;
  const int N = (int)p.N, R = (int)p.R, L = (int)p.L;
  const int n_first = wg.y * args.columns + 64 * wave, n_end = min(N, (wg.y + 1) * args.columns);
  const int id = token_id(p, args.up_tokens, m0, lane);

  for (int e = threadIdx.x; e < TOK * CH; e += 64 * kWaves) {
    const int c = e / CH, ch = e % CH, s = ch / 4;
    const bool there = c < args.up_tokens && m0 + c < p.M;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (there && 8 * ch < args.RP) {
      const float* from = args.part + (m0 + c) * args.RP + 8 * ch;
#pragma unroll 4
      for (int z = 0; z < args.splits; ++z) {
        const f32x4 u = *(const f32x4*)(from + (int64_t)z * p.M * args.RP);
        const f32x4 v = *(const f32x4*)(from + (int64_t)z * p.M * args.RP + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] += u[j];
          f[4 + j] += v[j];
        }
      }
    }
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(f[j]) < INFINITY ? fabsf(f[j]) : 0.f);
#pragma unroll
    for (int d = 1; d < CH; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    // the largest finite value to [2^kTop, 2^(kTop + 1))
    int e2 = (int)((__float_as_uint(top) >> 23) & 0xffu) - 127;
    e2 = top == 0.f ? 0 : min(max(e2, -112), 117);
    const float down = __uint_as_float((uint32_t)(127 + kTop - e2) << 23);
    u16x8 hi, lo, some;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float v[2] = {f[j] * down, f[j + 1] * down};
      const uint32_t both = toward_zero<DT>(v[0], v[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        hi[j + k] = (uint16_t)(both >> (16 * k));
        const float rest = v[k] - raw_at<DT>(Raw8<DT>{hi}, j + k);
        lo[j + k] = to16<DT>(rest == rest ? rest : 0.f);  // (infinity - infinity)
        some[j + k] = (uint16_t)min(__float_as_uint(f[j + k]) << 1, 1u);  // (0 for zeros)
      }
    }
    const u16x8 sign = hi & 0x8000;
    hi = sign | __builtin_elementwise_max((u16x8)(hi & 0x7fff), some);
    lo = sign | __builtin_elementwise_max((u16x8)(lo & 0x7fff), some);
    const int at = 16 * (ch % 4) + c % 16;
    low[c / 16][s][0][at] = hi;
    low[c / 16][s][1][at] = lo;
    if (ch == 0) {
      const int own = there ? p.ids[(uint32_t)(m0 + c) / (uint32_t)p.ids_rows] : -1;
      by[c] = make_float2(own >= 0 && own < L ? p.scaling[own] : 0.f, __uint_as_float((uint32_t)(127 - kTop + e2) << 23));
    }
  }
  __syncthreads();

  each_id(id, L, [&](int cur, uint64_t same) {
    const uint16_t* b = (const uint16_t*)p.b + (int64_t)cur * N * R;
    u16x8 bv[4][KS];
    auto fetch = [&](int n0) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int n = n0 + 32 * (t >> 1) + 8 * (col >> 2) + 4 * (t & 1) + (col & 3);
        const uint16_t* row = b + (int64_t)(n < N ? n : 0) * R;  // (columns past N are not kept)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int r = 32 * s + 8 * q;
          bv[t][s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
          if (r + 8 <= R) bv[t][s] = load8(row + r);
          else if (r < R) bv[t][s] = load_raw<DT>(row, r, R).v;
        }
      }
    };
    if (n_first < n_end) fetch(n_first);
    for (int n0 = n_first; n0 < n_end; n0 += 64 * kWaves) {
      const int at = n0 + 8 * q;
      const bool whole = n0 + 64 <= N;
      Raw8<DT> y[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if ((same >> (16 * t + col)) & 1) {
          const uint16_t* from = (const uint16_t*)p.y + (m0 + 16 * t + col) * p.y_stride;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (whole) y[t][k].v = load8(from + at + 32 * k);
            else if (at + 32 * k < N) y[t][k] = load_raw<DT>(from, at + 32 * k, N);
          }
        }
      u16x8 b0[4][KS];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int s = 0; s < KS; ++s) b0[t][s] = bv[t][s];
      if (n0 + 64 * kWaves < n_end) fetch(n0 + 64 * kWaves);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (!((same >> (16 * t)) & 0xffff)) continue;
        f32x4 acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const u16x8 hi = low[t][s][0][lane], lo = low[t][s][1][lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[i] = mfma16<DT>(b0[i][s], hi, acc[i]);
            acc[i] = mfma16<DT>(b0[i][s], lo, acc[i]);
          }
        }
        if ((same >> (16 * t + col)) & 1) {
          uint16_t* to = (uint16_t*)p.out + (m0 + 16 * t + col) * p.out_stride;
          const float2 w = by[16 * t + col];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = fmaf(w.x, w.y * acc[2 * k + (i >> 2)][i & 3], raw_at<DT>(y[t][k], i));
            if (at + 32 * k < N) store_raw<DT>(to, at + 32 * k, N, f);
          }
        }
      }
    }
  });

  // tokens without an adapter keep y, bit for bit: a wave takes every fourth of them, several rows in flight
  if (p.out == p.y) return;
  uint64_t left = __ballot(lane < args.up_tokens && m0 + lane < p.M && (id < 0 || id >= L));
  for (int skip = wave; skip; --skip) left &= left - 1;
  constexpr int ROWS = 4;
  while (left) {
    int64_t m[ROWS];
    int rows = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      m[i] = m0 + (left ? __builtin_ctzll(left) : 0);
      rows += left != 0;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) left &= left - 1;
    }
    for (int n = n_first - 64 * wave + 8 * lane; n < n_end; n += 8 * 64) {
      Raw8<DT> v[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (i < rows) v[i] = load_raw<DT>((const uint16_t*)p.y + m[i] * p.y_stride, n, n_end);
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if (i >= rows) continue;
        uint16_t* to = (uint16_t*)p.out + m[i] * p.out_stride;
        if (n + 8 <= n_end) *(u16x8_any*)(to + n) = v[i].v;
        else
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n + j < n_end) to[n + j] = v[i].v[j];
      }
    }
  }
}

// Few tokens with small adapters: one launch. A workgroup takes a token and 512
// of its columns, a thread each, and forms A x whole, again in each workgroup of
// the token (its eight waves a part of K each); B and y, which only the id is
// needed for, arrive meanwhile. Bound by A: a CU gets about 30 KB a us of it, so
// that the two launches, which read a part of it in each workgroup, win for
// large ones (us, kernels alone, one launch against two, which wait for each
// other as well): 64 tokens, 1024 to 1024, rank 16, 4.0 against 3.3 + 4.8; 50
// tokens, 1024 to 2048, rank 32, 5.3 against 3.7 + 4.6; 12 tokens, 4096 to 4096,
// rank 16, 7.4 against 3.4 + 5.6. Whole calls along the rule's product of rounds of
// the chip, rank and K, 12 tokens to 4096 columns: at 73728 (rank 16, K 4608) 7.7
// against 10.4, at 98304 (K 6144) 9.3 against 11.0; at 131072 they meet: 11.4
// against 11.7 (K 8192), 11.1 against 9.9 (rank 32, K 4096), 11.7 against 10.3
// (rank 16, K 4096, 11008 columns: two rounds); at rank 64 19 against 11. More
// steps of K under way: no change. RT: 16-row tiles of the rank.
constexpr int kOneWaves = 8, kOneColumns = 64 * kOneWaves, kOneRank = 32;

template <int DT, int RT>
__global__ __launch_bounds__(64 * kOneWaves) void adapter_one(const AdapterArgs args) {
  const actune_adapter_args& p = args.p;
  constexpr int AHEAD = 4;  // steps of K under way
  __shared__ float sums[kOneWaves][16 * RT];
  __shared__ __align__(16) float low[16 * RT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, q = lane >> 4;
  const int2 wg = item();
  const int m = wg.x, n = wg.y * kOneColumns + (int)threadIdx.x;
  const int K = (int)p.K, N = (int)p.N, R = (int)p.R;
  const int id = p.ids[(uint32_t)m / (uint32_t)p.ids_rows];
  const uint16_t* y = (const uint16_t*)p.y + m * p.y_stride;
  uint16_t* out = (uint16_t*)p.out + m * p.out_stride;
  const uint16_t y_n = y[min(n, N - 1)];
  if (id < 0 || id >= (int)p.L) {  // (the workgroup's one token)
    if (p.out != p.y && n < N) out[n] = y_n;
    return;
  }
  const float scaling = p.scaling[id];
  u16x8 b[2 * RT];
  const uint16_t* b_row = (const uint16_t*)p.b + ((int64_t)id * N + min(n, N - 1)) * R;
#pragma unroll
  for (int c = 0; c < 2 * RT; ++c) {
    b[c] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (8 * c + 8 <= R) b[c] = load8(b_row + 8 * c);
    else if (8 * c < R) b[c] = load_raw<DT>(b_row, 8 * c, R).v;
  }

  struct Step {
    u16x8 a[2][RT], x[2];
  };
  const uint16_t* x = (const uint16_t*)p.x + m * p.x_stride;
  const uint16_t* a[RT];
  f32x4 acc[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = 16 * i + col;
    a[i] = (const uint16_t*)p.a + ((int64_t)id * R + (r < R ? r : 0)) * K;  // (rows past the rank are not kept)
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto fetch = [&](Step& to, int k) {
    const int at = k + 8 * q;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      to.x[h] = load8(x + at + 32 * h);  // (every column of the product is this token)
#pragma unroll
      for (int i = 0; i < RT; ++i) to.a[h][i] = load8(a[i] + at + 32 * h);
    }
  };
  auto multiply = [&](const Step& of) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i] = mfma16<DT>(of.a[h][i], of.x[h], acc[i]);
  };
  constexpr int kStride = 64 * kOneWaves;
  const int first = 64 * wave, whole = max(0, (K - 63 - first + kStride - 1) / kStride);  // steps that do not pass K
  Step ring[AHEAD];
#pragma unroll
  for (int s = 0; s < AHEAD; ++s)
    if (s < whole) fetch(ring[s], first + s * kStride);
  int i0 = 0;
  for (; i0 + 2 * AHEAD <= whole; i0 += AHEAD)
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      multiply(ring[s]);
      fetch(ring[s], first + (i0 + s + AHEAD) * kStride);
    }
  for (; i0 < whole; i0 += AHEAD)
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
      if (i0 + s < whole) {
        multiply(ring[s]);
        if (i0 + s + AHEAD < whole) fetch(ring[s], first + (i0 + s + AHEAD) * kStride);
      }
  if (const int k = first + whole * kStride; k < K) {  // zeros past K's end
    const int at = k + 8 * q;
    const u16x8 none = {0, 0, 0, 0, 0, 0, 0, 0};
    Step end;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool any = at + 32 * h < K;
      end.x[h] = any ? load_raw<DT>(x, at + 32 * h, K).v : none;
#pragma unroll
      for (int i = 0; i < RT; ++i) end.a[h][i] = any ? load_raw<DT>(a[i], at + 32 * h, K).v : none;
    }
    multiply(end);
  }
  if (col == 0)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[wave][16 * i + 4 * q + e] = acc[i][e];
  __syncthreads();
  if (threadIdx.x < 16 * RT) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kOneWaves; ++w) s += sums[w][threadIdx.x];
    low[threadIdx.x] = (int)threadIdx.x < R ? s : 0.f;
  }
  __syncthreads();
  if (n >= N) return;
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < 2 * RT; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(raw_at<DT>(Raw8<DT>{b[c]}, j), low[8 * c + j], s);
  out[n] = to16<DT>(fmaf(scaling, s, raw_at<DT>(Raw8<DT>{u16x8{y_n}}, 0)));
}

struct Plan {
  int one;
  int RP, splits, chunk, down_tokens, up_tokens, columns;
};

// One launch or two (the workspace is the two launches' in either case), and the
// tokens, splits of K and columns of a workgroup.
//
// Tokens: up to 64 a workgroup takes one (in a decode step each has its own
// adapter, and the chip is filled by splits of K and columns), else 64 (32 for
// the second product of a rank above 64, whose operands leave no registers), or
// 16 where that leaves too few workgroups: fewer than two a CU down, one a CU up
// (500 tokens, 11008 columns, rank 16: 15.1 us with 64, 17.6 with 16; 800, 4096,
// rank 128: 15.7 with 32, 19.9 with 16; below it 1000, 2048, rank 32: 8.5 and
// 6.2).
//
// Splits, whole steps of the four waves (256 elements), at most 16: about two
// workgroups a CU; with 64 tokens the number with the least rounds of the chip,
// against the splits' sums that are written and read again (100 groups of rank
// 64: 42 us with three, 36 with four; 32 groups: 12 with eight, 13 with six).
// Fewer (408 tokens, K 4096, rank 16, four in place of 16) make up 8 us of 9 but
// down 6.6 of 4.
//
// Columns: two workgroups a CU (100 us, 106 with four; 8192 tokens, rank 64), four
// of 16 tokens (800 tokens, 4096 columns, rank 64: 12.7 us, 13.7 with two; 408
// tokens with one 12, with two 9.7).
Plan plan_of(int64_t M, int64_t N, int64_t K, int64_t R) {
  Plan g;
  g.RP = (int)((R + 15) / 16) * 16;
  const int64_t rounds = (M * ((N + kOneColumns - 1) / kOneColumns) + kCus - 1) / kCus;
  // (a grid's y stays below 2^16)
  g.one = M <= 64 && R <= kOneRank && rounds * g.RP * K <= 98304 && N <= kOneColumns * 65535;
  const int64_t steps = (K + 255) / 256, blocks = (N + 255) / 256;
  auto groups = [&](int64_t t) { return (M + t - 1) / t; };
  g.down_tokens = M <= 64 ? 1 : groups(16 * kDownTiles) * (steps < 16 ? steps : 16) < 2 * kCus ? 16 : 16 * kDownTiles;
  g.up_tokens = M <= 64 ? 1 : groups(16 * up_tiles(R)) * blocks < kCus ? 16 : 16 * up_tiles(R);
  const int64_t tiles = (M + g.down_tokens - 1) / g.down_tokens;
  int64_t splits = (2 * kCus + tiles - 1) / tiles;
  splits = splits < 1 ? 1 : splits;
  if (g.down_tokens > 16) {
    double least = -1;
    for (int s = 1; s <= 16; ++s) {
      const double t = (double)((tiles * s + kCus - 1) / kCus) / s + s * 0.5 * g.RP / K;
      if (least < 0 || t < least) {
        least = t;
        splits = s;
      }
    }
  }
  splits = splits > steps ? steps : splits > 16 ? 16 : splits;
  const int64_t per = (steps + splits - 1) / splits;
  g.chunk = (int)(per * 256);
  g.splits = (int)((steps + per - 1) / per);
  const int64_t rows = (M + g.up_tokens - 1) / g.up_tokens;
  int64_t cuts = ((g.up_tokens == 16 ? 4 : 2) * kCus + rows - 1) / rows;
  cuts = cuts < 1 ? 1 : cuts > blocks ? blocks : cuts;
  g.columns = (int)((blocks + cuts - 1) / cuts * 256);
  return g;
}

// (a dispatch holds less than 2^32 threads: 2^24 workgroups of up_tiles(R) 16s of tokens)
bool sizes_ok(int64_t M, int64_t N, int64_t K, int64_t R) {
  return M >= 0 && N > 0 && N <= INT_MAX / 2 && K > 0 && K <= INT_MAX / 2 && R > 0 && R <= kMaxRank &&
         M <= (int64_t)16 * up_tiles(R) * ((1 << 24) - 1);
}

template <int DT, int NT>
void launch_down(const AdapterArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.p.M + a.down_tokens - 1) / a.down_tokens), (unsigned)a.splits);
  if (a.RP <= 16) adapter_down<DT, 1, NT><<<grid, 64 * kWaves, 0, st>>>(a);
  else if (a.RP <= 32) adapter_down<DT, 2, NT><<<grid, 64 * kWaves, 0, st>>>(a);
  else adapter_down<DT, 4, NT><<<grid, 64 * kWaves, 0, st>>>(a);
}

template <int DT, bool MANY>
void launch_up(const AdapterArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.p.M + a.up_tokens - 1) / a.up_tokens), (unsigned)((a.p.N + a.columns - 1) / a.columns));
  if (a.RP <= 32) adapter_up<DT, 1, MANY ? up_tiles(32) : 1><<<grid, 64 * kWaves, 0, st>>>(a);
  else if (a.RP <= 64) adapter_up<DT, 2, MANY ? up_tiles(64) : 1><<<grid, 64 * kWaves, 0, st>>>(a);
  else adapter_up<DT, 4, MANY ? up_tiles(128) : 1><<<grid, 64 * kWaves, 0, st>>>(a);
}

template <int DT>
void launch_one(const AdapterArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.p.M, (unsigned)((a.p.N + kOneColumns - 1) / kOneColumns));
  if (a.RP <= 16) adapter_one<DT, 1><<<grid, 64 * kOneWaves, 0, st>>>(a);
  else adapter_one<DT, 2><<<grid, 64 * kOneWaves, 0, st>>>(a);
}

template <int DT>
void launch_adapter(const AdapterArgs& a, hipStream_t st) {
  if (a.down_tokens <= 16) launch_down<DT, 1>(a, st);
  else launch_down<DT, kDownTiles>(a, st);
  if (a.up_tokens <= 16) launch_up<DT, false>(a, st);
  else launch_up<DT, true>(a, st);
}

}  // namespace
}  // namespace actune

using namespace actune;

extern "C" {

int64_t actune_adapter_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t R) {
  if (!sizes_ok(M, N, K, R)) return -1;
  if (M == 0) return 0;
  const Plan g = plan_of(M, N, K, R);
  return (int64_t)g.splits * M * g.RP * 4;
}

int actune_adapter_add(const actune_adapter_args* args, void* stream) {
  block_clear_error();
  if (!args) return block_fail("null pointer");
  const actune_adapter_args& p = *args;
  if (p.dtype != kBF16 && p.dtype != kF16) return block_fail("adapters take bf16 or f16");
  if (p.R < 1 || p.R > kMaxRank) return block_fail("rank must be between 1 and 128");
  if (!sizes_ok(p.M, p.N, p.K, p.R) || p.L < 0 || p.L > INT_MAX) return block_fail("invalid dimensions");
  const int64_t most = INT64_MAX / 4 / (p.M + 1);
  for (int64_t s : {p.x_stride, p.y_stride, p.out_stride})
    if (s < 0 || s > most) return block_fail("invalid row stride");
  if (p.ids_rows < 1 || p.ids_rows > INT_MAX) return block_fail("an id covers one row at least");
  if (p.out_stride < p.N && p.M > 1) return block_fail("rows of out overlap");
  // (its rows would be written where others of y are yet to be read)
  if (p.out && p.out == p.y && p.out_stride != p.y_stride && p.M > 1) return block_fail("out on y needs y's row stride");
  if (p.M == 0) return kOk;
  if (!p.x || !p.y || !p.ids || !p.out || (p.L > 0 && (!p.a || !p.b || !p.scaling))) return block_fail("null pointer");
  const Plan g = plan_of(p.M, p.N, p.K, p.R);
  if (!p.workspace || p.workspace_bytes < (int64_t)g.splits * p.M * g.RP * 4) return block_fail("workspace too small");
  for (const void* t : {p.x, p.y, p.a, p.b, (const void*)p.out})
    if (!is_aligned(t, 2)) return block_fail("misaligned operand");
  if (!is_aligned(p.scaling, 4) || !is_aligned(p.ids, 4) || !is_aligned(p.workspace, 16))
    return block_fail("misaligned operand");
  const AdapterArgs a{p, (float*)p.workspace, g.RP, g.splits, g.chunk, g.down_tokens, g.up_tokens, g.columns};
  // (in one launch a workgroup writes columns of out while another reads the token's x)
  const uintptr_t x0 = (uintptr_t)p.x, out0 = (uintptr_t)p.out;
  const bool apart = x0 + 2 * ((p.M - 1) * p.x_stride + p.K) <= out0 ||
                     out0 + 2 * ((p.M - 1) * p.out_stride + p.N) <= x0;
  if (g.one && apart) {
    if (p.dtype == kBF16) launch_one<kBF16>(a, (hipStream_t)stream);
    else launch_one<kF16>(a, (hipStream_t)stream);
  } else if (p.dtype == kBF16) launch_adapter<kBF16>(a, (hipStream_t)stream);
  else launch_adapter<kF16>(a, (hipStream_t)stream);
  return block_status();
}

}  // extern "C"
