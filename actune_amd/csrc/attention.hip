// Attention of a batch of sequences over a prefix that they share and keys of
// their own:
//
//   out = sum_j softmax(scale q . k_j) v_j,  lse = log sum_j exp(scale q . k_j)
//
// One pass over the keys with a running maximum and sum. Scores are formed
// transposed, S^T = K Q^T in 32 x 32 MFMA tiles: a lane then holds 16 scores of
// ONE query, so that the maximum, the sum and the rescaling of the output
// (O^T = V^T P^T, the same lane the same query) need no exchange beyond the two
// halves of the wave, and the rounded P^T registers are the next product's
// operand as they stand. That operand's keys come in the order 4h..4h+3,
// 8+4h..8+4h+3 of each 16; a sum has no order, so V is read in the same one,
// transposed out of LDS by the hardware.
//
// K and V tiles go to LDS by DMA loads, tiles ahead of their use. The 16-byte
// chunks of a tile row are permuted by row, so that both the row reads of K and
// the transposed reads of V spread over all banks; the DMA writes LDS in lane
// order, hence the source addresses carry the permutation.
//
// Row tiles, items and parts. The rows of one key head are T queries by
// Hq / Hkv heads of one sequence (joint: its tile goes over the prefix and its
// own keys in one sweep), or those of every sequence of the group side by side
// (stacked: the prefix is swept once for all of them, the own keys are items of
// their own). A sweep is cut into splits where there are too few tiles for the
// chip. Each (tile, split) leaves output and statistics in the workspace, and
// a second launch joins the parts; one part alone writes the output itself.
//
// Measured (bf16, kernel and, where there are parts, join):
//   8 prompts of 512 behind 2050 keys, 32 heads of 128, causal: 190 us, 0.82
//     PFLOP/s (a library product of 8192^3 here: 1.19). The matrix units are
//     busy 39 percent of the cycles, the vector units issue in 45: a wave's tile
//     goes through products, exponentials and products, and the two waves a SIMD
//     overlap only in part.
//   32 chunks of 50, 8 heads of 256 over one, 768 keys seen of 968 and 50: 34.4
//     + 7.0 us, 0.31 PFLOP/s. Each workgroup sweeps 9 tiles (20 us), those that
//     the mask empties among them; the rest is its start, 26 MB of parts, and
//     reading them again.
//   24 requests, 32 heads of 128, 4096 keys and 160: 31 + 4.7 us for 114 MB.
//     Bound by the own keys' items, whose loads are a few tiles deep.
//   48 requests, 8 heads of 256 over one, 65537 keys and 300 (f16): 53 + 8.0 us,
//     78 MB and 26 GFLOP. Bound by its cut: 159 workgroups sweep 20 tiles of 64
//     keys each, 2.3 us a tile, beside 96 with two or three tiles of own keys
//     (own keys in one item each leave room for 240 with 15 tiles: 45 + 9.0).
//   one request, 8 heads of 128 read by 32, 65536 keys: 45 us, 268 MB, 5.9 TB/s.
//   one chunk of 50, 816 keys: 12.1 + 4.0 us, most of it two launches' latency.
//
// The probabilities are rounded to the operands' type for the second product,
// their sum is not. That is where the outputs' error comes from beside their own
// rounding: 0.0022 of the 2-norm in bf16 (f32 probabilities: 0.0017), 0.00028 in
// f16 (0.00021), where many keys count. A second 16-bit part of them takes it
// away for half as many products again: 242 us for the 190 of the prompts, 39.2
// for 37.5 a call of the 24 requests, 15.9 for 15.4 of the one chunk; the wave
// pairs have no LDS for it. One part in every form, so that the precision does
// not depend on the layout.
#include <climits>
#include <cmath>

#include "block.hpp"
#include "launch.hpp"

namespace actune {
namespace {

constexpr int kTileRows = 128, kSmallRows = 32;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Division of 0 <= n < 2^31 by a number known before the launch: with 2^s the
// power of two at or above d, m = floor(2^32 (2^s - d) / d) + 1 gives n / d =
// (hi(n m) + n) >> s.
struct Div {
  uint32_t d, m, s;
};
Div div_of(int64_t d) {
  Div r{(uint32_t)d, 0, 0};
  while (((uint64_t)1 << r.s) < (uint64_t)d) ++r.s;
  r.m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << r.s) - d)) / d + 1);
  return r;
}
__device__ __forceinline__ int quotient(int n, const Div& d) {
  return (int)((__umulhi((uint32_t)n, d.m) + (uint32_t)n) >> d.s);
}
// n := n / d, returning the remainder
__device__ __forceinline__ int take(int& n, const Div& d) {
  const int q = quotient(n, d), r = n - q * (int)d.d;
  n = q;
  return r;
}

// Tiles of keys cut into splits: split i starts at i * per + min(i, extra).
struct Cut {
  int per, extra;
};
Cut cut_of(int64_t tiles, int64_t splits) { return Cut{(int)(tiles / splits), (int)(tiles % splits)}; }
__device__ __forceinline__ int start_of(const Cut& c, int i) { return i * c.per + min(i, c.extra); }

struct Plan {
  int big;            // row tiles of 128 (else 32)
  int stacked;        // rows of a whole group side by side
  int tiles;          // row tiles of a main item's row set
  int splits;         // key splits of the main items
  int own_tiles;      // row tiles and key splits of the own-key items (stacked)
  int own_splits;
  int parts;          // parts of a row
  int64_t pre_cap, own_cap;  // tiles of the prefix and of a sequence's own keys
  int64_t main_items, own_items;
};

struct AttnArgs {
  actune_prefix_attention_args p;
  int parts, splits;
  int main_items;
  int first;            // the launch's first item or, of a join, row
  int pre_cap;          // tiles of the prefix
  int per_group;        // sequences of a group
  int set_rows;         // rows of a main item's row set, and of one sequence's
  int seq_rows;
  Div tiles, per_group_div, splits_div, heads, own_tiles, own_splits, rows, share;
  Cut cut, own_cut;
  float factor;         // scale * log2(e)
  float* part_o;        // [parts][B T Hq][DP]
  float* part_ml;       // [parts][B T Hq][2]: maximum (log2 units) and sum
};

// f16 keeps small probabilities out of its subnormals: they are scaled by 2^7
// (with the 2^8 that a maximum may lag behind, below 2^16); the factor leaves
// with the sum.
template <int DT>
__device__ __forceinline__ constexpr float lift() { return DT == kF16 ? 7.f : 0.f; }

// two values to the 16-bit type, a in the low half
template <int DT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == kBF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

template <int DT>
__device__ __forceinline__ f32x16 mfma32(u16x8 a, u16x8 b, f32x16 c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 16 bytes of each lane from base + voff to LDS at m0 + 16 lane. Issued from
// inline asm, which the compiler's wait counts do not follow: it would wait for
// every load in flight before any LDS read. The kernel waits for them itself;
// the waits and barriers are what orders LDS accesses around them.
__device__ __forceinline__ void dma16(const void* base, uint32_t voff, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0), "v"(voff), "s"(base) : "m0");
}
// the same from an address of each lane's own
__device__ __forceinline__ void dma16(const void* from, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(m0), "v"(from) : "m0");
}
// all but the N youngest loads of this wave have arrived, and every LDS access
// before has been done
template <int N = 0>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Chunk c of tile row r sits at chunk c ^ swizzle(r). A row read of K takes one
// chunk of 16 consecutive rows at a time, a transposed read of V 64 bytes of
// four: the low two row bits pick the 64-byte group, the next two the chunk in
// it, so that either covers all banks once (rows of 128 bytes: two rows lie
// side by side, one bit less picks the group).
template <int DP>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (DP == 64) return 4 * ((r >> 1) & 1) + ((r >> 2) & 3);
  else return 4 * (r & 3) + ((r >> 2) & 3);
}

// A run of keys: the prefix of a group or a sequence's own, for one key head.
struct Keys {
  const uint16_t* k;
  const uint16_t* v;
  uint32_t k_bytes, v_bytes;  // token strides
  const uint8_t* mask;        // or nullptr
  int end;                    // keys that exist
};

__device__ const v4u kZeros = {0, 0, 0, 0};

// DMA loads of tiles of KT rows, BLOCKS KiB of each by a wave: block i holds
// rows (wave BLOCKS + i) 512 / DP on. Rows past the end read the last row that
// exists (their scores are masked and their values cleared).
template <int DP, int KT, int WAVES>
struct Loader {
  static constexpr int BLOCKS = KT * DP * 2 / 1024 / WAVES, RPB = 512 / DP;
  static_assert(KT * DP * 2 % (1024 * WAVES) == 0, "whole blocks");
  int row;        // this lane's row in block 0
  uint32_t chunk; // byte offset of its chunk there; block i's differs by a constant's bits (the rows' bits do not overlap)
  uint32_t lds;   // of the wave's block 0
  uint32_t origin;
  uint32_t width; // bytes of a row's D columns
  __device__ __forceinline__ Loader(int D, int wave, uint32_t lds0) {
    const int lane = threadIdx.x & 63;
    row = wave * BLOCKS * RPB + lane / (DP / 8);
    origin = lds0;
    lds = __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)wave * BLOCKS * 1024);
    chunk = 16 * ((lane % (DP / 8)) ^ swizzle<DP>(row));
    width = 2 * D;
  }
  struct Tile {
    const uint8_t* base;
    uint32_t stride;  // below 2^24
    int last;         // last row that exists
    uint32_t at;      // place in LDS
  };
  static __device__ __forceinline__ Tile tile(const uint16_t* src, uint32_t stride, int first, int end, uint32_t at) {
    const int row0 = min(first, end - 1);  // in range also where the whole tile lies past the end
    return Tile{(const uint8_t*)src + (uint64_t)(uint32_t)row0 * stride, stride, end - 1 - row0, at};
  }
  __device__ __forceinline__ uint32_t column(int i) const { return chunk ^ (16 * swizzle<DP>(i * RPB)); }
  // Keys: columns past D are zeros, as those of q are (an infinity there would make the score NaN). A wave with few
  // blocks leaves out the lanes that stand for them, whose places clear_columns has written; one that loads a whole
  // tile reads zeros instead, since clearing 32 blocks takes 1 us of a short call (8 prompts of 512, 12 heads of 80,
  // 2050 keys: 85 us without the lanes, 89.5 with zeros; a chunk of 50, 8 heads of 200, 816 keys: 16.1 and 15.1).
  static constexpr bool ZEROS = WAVES == 1;
  __device__ __forceinline__ void request_keys(const Tile& t) const {
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      const uint32_t c = column(i), from = __umul24((uint32_t)min(row + i * RPB, t.last), t.stride) + c;
      if (ZEROS && width < 2 * DP) dma16(c < width ? t.base + from : (const uint8_t*)&kZeros, lds + t.at + i * 1024);
      else if (c < width) dma16(t.base, from, lds + t.at + i * 1024);
    }
  }
  // zeros past D in this wave's blocks of the place at `to`
  __device__ __forceinline__ void clear_columns(uint8_t* to) const {
    if (ZEROS || width == 2 * DP) return;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
      if (column(i) >= width) *(u16x8*)(to + i * 1024 + 16 * (threadIdx.x & 63)) = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
  // Values: past D any data of the row, in columns that are not stored.
  __device__ __forceinline__ void request_values(const Tile& t) const {
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      const uint32_t c = column(i);
      dma16(t.base, __umul24((uint32_t)min(row + i * RPB, t.last), t.stride) + (c < width ? c : 0), lds + t.at + i * 1024);
    }
  }
};

// Order of N products that take READS LDS reads each: a few reads ahead, then
// one product and the reads of a later one in turn. Left to itself the compiler
// waits for each read where it is used.
template <int N, int READS>
__device__ __forceinline__ void feed() {
  constexpr int AHEAD = N < 4 ? N : 4;
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x8, AHEAD, 0);
}

// A lane's query: row r of the row set of a key head (one sequence's, or a whole
// group's where stacked), live below `end`.
struct Row {
  bool live;
  int t;
  int out;              // its row of out and lse
  const uint16_t* q;
};
template <bool STACKED>
__device__ __forceinline__ Row row_of(const AttnArgs& args, int group_or_seq, int head, int r, int end) {
  const actune_prefix_attention_args& p = args.p;
  const bool live = r < end;
  int seq = live ? r : 0;  // (the others read what row 0 reads, and write nothing)
  const int rs = STACKED ? take(seq, args.rows) : seq;
  const int t = quotient(rs, args.share), hq = head * (int)args.share.d + rs - t * (int)args.share.d;
  const int64_t b = STACKED ? (int64_t)group_or_seq * args.per_group + seq : group_or_seq;
  return Row{live, t, (int)((b * p.T + t) * p.Hq + hq),
             (const uint16_t*)p.q + b * p.q_stride[0] + t * p.q_stride[1] + hq * p.q_stride[2]};
}

// Operand fragments of a lane's query (half h of each 16 columns), zeros past D,
// from memory: 32 rows a load, which costs the address path 32 lines; for few
// rows.
template <int DP>
__device__ __forceinline__ void load_query(const Row& row, int D, int h, u16x8 (&qf)[DP / 16]) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) qf[s] = *(const u16x8*)(row.q + min(16 * s + 8 * h, D - 8));
  // arrived here: inside a loop the compiler's wait for them would be one for every load in flight
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) asm volatile("" : "+v"(qf[s]));
  if (D < DP) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
      if (16 * s + 8 * h >= D) qf[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
}

// The infinities and NaN among eight values, the others as zeros.
template <int DT>
__device__ __forceinline__ u16x8 strange_of(u16x8 v) {
  constexpr uint16_t kInf = DT == kBF16 ? 0x7f80 : 0x7c00;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (v[e] & kInf) == kInf ? v[e] : 0;
  return v;
}
// Causal hides keys of a tile from some queries and shows them to others: their
// infinite and NaN values, which a probability of 0 would make NaN, leave the
// tile, and add_strange adds them to the sums of the queries that see them.
// Returns whether there were any.
template <int DT, int DP, int KT>
__device__ __forceinline__ bool take_strange(uint8_t* vt, int at, int threads) {
  bool any = false;
#pragma unroll 1
  for (int c = at; c < KT * DP / 8; c += threads) {
    u16x8* const to = (u16x8*)(vt + 16 * c);
    const u16x8 v = *to, s = strange_of<DT>(v);
    const v4u bits = __builtin_bit_cast(v4u, s);
    if (bits[0] | bits[1] | bits[2] | bits[3]) {
      any = true;
      *to = v ^ s;
    }
  }
  return any;
}
// Keys whose strange values were taken out: `first` .. last - 1.
struct Taken {
  const uint16_t* v;
  uint32_t v_bytes;
  int first, last;
};
// Those of a key's columns d .. d + 3.
template <int DT>
__device__ __forceinline__ f32x4 strange_at(const Taken& from, int key, int d) {
  const u16x4 v = *(const u16x4*)((const uint8_t*)from.v + (uint64_t)(uint32_t)key * from.v_bytes + 2 * d);
  u16x8 w = {v[0], v[1], v[2], v[3], 0, 0, 0, 0};
  w = strange_of<DT>(w);
  return f32x4{raw_at<DT>(Raw8<DT>{w}, 0), raw_at<DT>(Raw8<DT>{w}, 1), raw_at<DT>(Raw8<DT>{w}, 2), raw_at<DT>(Raw8<DT>{w}, 3)};
}

// A row's statistics: its part's, or lse where the part is the whole.
template <int DT>
__device__ __forceinline__ void write_stats(const AttnArgs& args, int64_t out_row, int part, float m, float l) {
  const actune_prefix_attention_args& p = args.p;
  if (args.parts == 1) {
    // sums over lifted probabilities: the log takes the lift back
    if (p.lse) p.lse[out_row] = l == 0.f ? -INFINITY : (m - lift<DT>() + __builtin_log2f(l)) * 0.693147180559945309f;
  } else {
    float* ml = args.part_ml + 2 * ((int64_t)part * p.B * p.T * p.Hq + out_row);
    // (a NaN sum without a maximum has to reach the join)
    ml[0] = l == 0.f ? -INFINITY : m == -INFINITY ? 0.f : m;
    ml[1] = l;
  }
}

// Columns d0 .. d0 + 32 N - 1 of a row, from N blocks of O^T (a lane holds 4 of
// each 8 columns).
template <int DT, int DP, int N>
__device__ __forceinline__ void write_out(const AttnArgs& args, int64_t out_row, int part, const f32x16* acc, int d0,
                                          int h, float l) {
  const actune_prefix_attention_args& p = args.p;
  const int D = (int)p.D;
  const bool direct = args.parts == 1;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float* po = args.part_o + ((int64_t)part * p.B * p.T * p.Hq + out_row) * DP;
  uint16_t* out = (uint16_t*)p.out + out_row * D;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int d = d0 + 32 * i + 8 * k + 4 * h;
      if (d0 + 32 * i + 8 * k >= D) continue;  // (whole eights: the same for every lane)
      if (direct) {
        u16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to16<DT>(acc[i][4 * k + e] * inv);
        *(u16x4*)(out + d) = v;
      } else {
        *(f32x4*)(po + d) = f32x4{acc[i][4 * k], acc[i][4 * k + 1], acc[i][4 * k + 2], acc[i][4 * k + 3]};
      }
    }
}

// The same for 32 rows of a wave through 8 KiB of LDS of its own, 64 columns at
// a time, so that stores cover whole lines (straight from the registers each
// touches 32 rows, which took a workgroup of heads of 256 5000 cycles). `out`:
// this lane's row (lanes 0 .. 31), negative where it is not live; `seen`: the
// own keys that it sees.
template <int DT, int DP, int N>
__device__ __forceinline__ void write_rows(const AttnArgs& args, uint8_t* lds, int out, int part, const f32x16* acc,
                                           int d0, float l, const Taken& from, int seen) {
  const actune_prefix_attention_args& p = args.p;
  const int lane = threadIdx.x & 63, q = lane & 31, h = lane >> 5, D = (int)p.D;
  const bool direct = args.parts == 1;
  const float by = !direct ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < N / 2; ++c) {
    const int d1 = d0 + 64 * c;
    if (d1 >= D) break;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[2 * c + i][4 * k + e] * by;
        *(f32x4*)(lds + q * 256 + 16 * ((8 * i + 2 * k + h) ^ (q & 15))) = v;
      }
    if (__any(seen > from.first)) {
#pragma unroll 1
      for (int t = 0; t < 8; ++t) {
        const int r = 4 * t + (lane >> 4), d = d1 + 4 * (lane & 15), last = min(__shfl(seen, r), from.last);
        f32x4* const at = (f32x4*)(lds + r * 256 + 16 * ((lane & 15) ^ (r & 15)));
        f32x4 v = *at;
#pragma unroll 1
        for (int key = from.first; key < last; ++key)
          if (d < D) v += strange_at<DT>(from, key, d);
        *at = v;
      }
    }
    if (direct) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int r = 8 * t + (lane >> 3), col = 8 * (lane & 7);
        const int to = __shfl(out, r);
        float f[8];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f32x4 v = *(const f32x4*)(lds + r * 256 + 16 * ((2 * (lane & 7) + k) ^ (r & 15)));
#pragma unroll
          for (int e = 0; e < 4; ++e) f[4 * k + e] = v[e];
        }
        if (to >= 0 && d1 + col < D) store_raw<DT>((uint16_t*)p.out + (int64_t)to * D, d1 + col, D, f);
      }
    } else {
      float* po = args.part_o + (int64_t)part * p.B * p.T * p.Hq * DP;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int r = 4 * t + (lane >> 4), col = 4 * (lane & 15);
        const int to = __shfl(out, r);
        const f32x4 v = *(const f32x4*)(lds + r * 256 + 16 * ((lane & 15) ^ (r & 15)));
        if (to >= 0 && d1 + col < D) *(f32x4*)(po + (int64_t)to * DP + d1 + col) = v;
      }
    }
  }
}

// Keys of a tile that a query sees, as bits, for the 32 keys from bit 32 u on
// and a lane's half h: bit 8 (i / 4) + i % 4 is score i's.
__device__ __forceinline__ uint32_t half_bits(uint64_t bits, int u, int h) { return (uint32_t)(bits >> (32 * u)) >> (4 * h); }
__device__ __forceinline__ void hide(f32x16& sc, uint32_t w) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!((w >> (8 * (i >> 2) + (i & 3))) & 1)) sc[i] = -INFINITY;
}

// Clears the rows of a V tile whose bit is not set (what stands at masked
// places may be NaN, and 0 * NaN is NaN); thread `at` of `threads`.
template <int DP, int KT>
__device__ __forceinline__ void clear_rows(uint8_t* vt, uint64_t bits, int at, int threads) {
  for (int c = at; c < KT * DP / 8; c += threads)
    if (!((bits >> (c / (DP / 8))) & 1)) *(u16x8*)(vt + 16 * c) = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
}

// The new running maximum of a query where its scores' maximum `top` (log2
// units) is far enough above the old one, and the factor of what has been
// summed. It may lag by 2^kLag: then nothing is rescaled.
constexpr float kLag = 8.f;
__device__ __forceinline__ float raise(float& m, float top) {
  const float to = fmaxf(m, top);
  const float by = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
  m = to;
  return by;
}

// What a workgroup sweeps: na tiles of `pre` from tile a0, then nb of `own` from
// b0, for the rows row0 .. end - 1 of a row set (its tile's number of them).
struct Item {
  Keys pre, own;
  int a0, na, b0, nb;
  int group_or_seq, head, row0, end, part;
  int low;  // the first own key that causal hides from some query
  // whether it hides keys of the own tile that starts at `first`
  __device__ __forceinline__ bool divides(int first, int kt) const { return min(first + kt, own.end) > low; }
  // the keys of all such tiles of kt keys (of an item's of `step`)
  __device__ __forceinline__ Taken taken(int kt, int step) const {
    return Taken{own.v, own.v_bytes, max(max(low, 0) / kt * kt, b0 * step), min((b0 + nb) * step, own.end)};
  }
};

template <int DP>
__device__ __forceinline__ uint32_t value_place(int r, int c) {
  return r * DP * 2 + 16 * ((c >> 3) ^ swizzle<DP>(r)) + 2 * (c & 7);
}
// Places of a wave's reads in a tile. A row starts at a multiple of its size, so
// that the chunk's permutation and the step are both xors of the place: one
// register and a constant for each read. opaque() keeps the compiler from
// holding all of them over the loop instead, which cost the pairs' kernel 20
// registers that it does not have.
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}
// K: row (lane % 32) of 32, half h of each 16 columns; step st of the columns at ^ 32 st.
template <int DP>
__device__ __forceinline__ uint32_t key_place() {
  const int lane = threadIdx.x & 63, r = lane & 31;
  return opaque(r * DP * 2 + 16 * ((lane >> 5) ^ swizzle<DP>(r)));
}
// V^T operand of 16 keys and columns c0 .. c0 + 31 (lane's: c0 + lane % 32), keys
// in the order of the probabilities' registers: two transposed reads, rows 8
// apart; columns 32 i on at ^ 64 i.
struct ValuePlace {
  uint32_t a, b;
};
template <int DP>
__device__ __forceinline__ ValuePlace value_places(int c0) {
  const int lane = threadIdx.x & 63;
  const int r = 4 * (lane >> 5) + ((lane & 15) >> 2), c = c0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  return ValuePlace{opaque(value_place<DP>(r, c)), opaque(value_place<DP>(r + 8, c))};
}
template <int DP>
__device__ __forceinline__ u16x8 value_frag(const uint8_t* vt, const ValuePlace& at, int k, int i) {
  typedef __attribute__((address_space(3))) s16x4* Lds;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(vt + (at.a ^ (64 * i)) + 16 * k * DP * 2));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(vt + (at.b ^ (64 * i)) + 16 * k * DP * 2));
  return __builtin_bit_cast(u16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
// Scores of 32 keys from row r0 of a K tile: a lane's 16 of query lane % 32.
template <int DT, int DP>
__device__ __forceinline__ f32x16 score_tile(const uint8_t* kt, int r0, const u16x8 (&qf)[DP / 16]) {
  const uint32_t at = key_place<DP>();
  f32x16 sc;
#pragma unroll
  for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
  for (int st = 0; st < DP / 16; ++st)
    sc = mfma32<DT>(*(const u16x8*)(kt + (at ^ (32 * st)) + r0 * DP * 2), qf[st], sc);
  return sc;
}
// The wait states before the first read of scores: the compiler leaves too few
// where the read comes behind a branch.
__device__ __forceinline__ void settle(f32x16& a, f32x16& b) { asm volatile("s_nop 11" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void settle(f32x16& a) { asm volatile("s_nop 11" : "+v"(a)); }

__device__ __forceinline__ float highest(const f32x16& sc, float top) {
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[i]);
  return top;
}
// the two halves' values joined (the lanes of a query), in both
__device__ __forceinline__ float2 halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_halves(float v) {
  const float2 r = halves(v);
  return fmaxf(r.x, r.y);
}
__device__ __forceinline__ float sum_halves(float v) {
  const float2 r = halves(v);
  return r.x + r.y;
}

// Probabilities of 16 scores as two operand fragments; their sum is added to l.
template <int DT>
__device__ __forceinline__ void probabilities(const f32x16& sc, float factor, float less, u16x8* pf, float& l) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float e = __builtin_amdgcn_exp2f(fmaf(sc[i], factor, -less));
    sum += e;
    pf[i >> 3][i & 7] = to16<DT>(e);
  }
  l += sum;
}
// Scores of the next tile in nx while the probabilities of this one are formed
// from sc: after each product one LDS read of a later one and the exponentials
// that its time covers, an order that the compiler does not find (it forms the
// probabilities where they are used) and is held to.
template <int DT, int DP, int SU>
__device__ __forceinline__ void scores_beside(const uint8_t* kt, int r0, const u16x8 (&qf)[DP / 16], f32x16 (&nx)[SU],
                                              const f32x16 (&sc)[SU], float factor, float less, u16x8 (&pf)[2 * SU],
                                              float& l) {
  constexpr int STEPS = DP / 16, N = SU * STEPS, RING = 4;
  const uint32_t at = key_place<DP>();
  auto key = [&](int i) {
    return *(const u16x8*)(kt + (at ^ (32 * (i % STEPS))) + (r0 + 32 * (i / STEPS)) * DP * 2);
  };
  u16x8 kf[RING];
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) kf[i] = key(i);
#pragma unroll
  for (int u = 0; u < SU; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) nx[u][i] = 0.f;
  uint32_t packed[8 * SU];
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    nx[i / STEPS] = mfma32<DT>(kf[i % RING], qf[i % STEPS], nx[i / STEPS]);
    if (i + RING - 1 < N) kf[(i + RING - 1) % RING] = key(i + RING - 1);
    // two at a time: a packed conversion each
#pragma unroll
    for (int e = 16 * i / STEPS / 2 * 2; e < 16 * (i + 1) / STEPS / 2 * 2; e += 2) {
      const float a = __builtin_amdgcn_exp2f(fmaf(sc[e / 16][e % 16], factor, -less));
      const float b = __builtin_amdgcn_exp2f(fmaf(sc[e / 16][e % 16 + 1], factor, -less));
      sum[0] += a;
      sum[1] += b;
      uint32_t both = pack16<DT>(a, b);
      asm volatile("" : "+v"(both));
      packed[e / 2] = both;
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  l += sum[0] + sum[1];
#pragma unroll
  for (int k = 0; k < 2 * SU; ++k)
    pf[k] = __builtin_bit_cast(u16x8, v4u{packed[4 * k], packed[4 * k + 1], packed[4 * k + 2], packed[4 * k + 3]});
}

// Scores of keys that a query does not see: those without a bit, and own keys
// from the query's limit on (`open` keys of the tile lie before it).
template <int KT, int N>
__device__ __forceinline__ void mask_scores(f32x16 (&sc)[N], uint64_t bits, int open, int u0, int h) {
  constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
  if (bits == kAll && !__any(open < KT)) return;
  if (open < KT) bits &= open <= 0 ? 0 : (1ull << open) - 1;
#pragma unroll
  for (int u = 0; u < N; ++u) hide(sc[u], half_bits(bits, u0 + u, h));
}

// Few rows: WK waves take the tile's rows (32) each, and 32 keys of each tile of
// 32 WK in LDS of their own, two stages, without a barrier; their parts join in
// LDS at the end. Bound by the keys' bytes.
template <int DP, int WK>
struct Small {
  static constexpr int TILE = 32 * DP * 2, STAGE = 2 * TILE, LDS = 2 * STAGE * WK;
};

template <int DT, int DP, int WK, bool STACKED, bool FULL>
__device__ __forceinline__ void sweep_small(const AttnArgs& args, uint8_t* lds, const Item& it) {
  using G = Small<DP, WK>;
  constexpr int OB = DP / 32;
  const actune_prefix_attention_args& p = args.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane & 31, h = lane >> 5;
  const int D = FULL ? DP : (int)p.D;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * 2 * G::STAGE;
  uint8_t* const mem = lds + wave * 2 * G::STAGE;
  const Loader<DP, 32, 1> loader(D, 0, base);
  using L = Loader<DP, 32, 1>;
  const int n = it.na + it.nb;
  auto first_of = [&](int j) { return ((j < it.na ? it.a0 + j : it.b0 + j - it.na) * WK + wave) * 32; };
  uint32_t there = 0;  // lane i: whether key i of the tile requested last exists and is not masked
  auto request = [&](int j) {
    const bool in_pre = j < it.na;
    const Keys& s = in_pre ? it.pre : it.own;
    const int first = first_of(j), key = first + lane;
    there = lane < 32 && key < s.end;
    if (there && s.mask) there = s.mask[key];  // (used a tile later: nothing waits here)
    loader.request_keys(L::tile(s.k, s.k_bytes, first, s.end, (j & 1) * G::STAGE));
    loader.request_values(L::tile(s.v, s.v_bytes, first, s.end, (j & 1) * G::STAGE + G::TILE));
  };
  if (n > 0) request(0);
  const Row row = row_of<STACKED>(args, it.group_or_seq, it.head, it.row0 + q, it.end);
  u16x8 qf[DP / 16];
  load_query<DP>(row, D, h, qf);
  f32x16 acc[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
  float m = -INFINITY, l = 0.f;
  // the first own key that causal hides from this query
  const int limit = p.causal ? it.own.end - (int)p.T + row.t + 1 : INT_MAX;
  bool strange = false;

  for (int j = 0; j < n; ++j) {
    wait_loads();
    const uint64_t bits = __ballot(there != 0);
    if (j + 1 < n) request(j + 1);
    uint8_t* const kt = mem + (j & 1) * G::STAGE;
    uint8_t* const vt = kt + G::TILE;
    if (bits == 0) continue;
    if (bits != 0xffffffffull) clear_rows<DP, 32>(vt, bits, lane, 64);
    if (j >= it.na && it.divides(first_of(j), 32) && __any(take_strange<DT, DP, 32>(vt, lane, 64))) strange = true;
    f32x16 sc[1] = {score_tile<DT, DP>(kt, 0, qf)};
    feed<DP / 16, 1>();
    settle(sc[0]);
    mask_scores<32>(sc, bits, j < it.na ? INT_MAX : limit - first_of(j), 0, h);
    float top = highest(sc[0], -INFINITY);
    top = max_halves(top) * args.factor;
    if (__any(top > m + kLag)) {
      const float by = raise(m, top);
      l *= by;
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[i][k] *= by;
    }
    u16x8 pf[2];
    probabilities<DT>(sc[0], args.factor, m == -INFINITY ? 0.f : m - lift<DT>(), pf, l);
    const ValuePlace at = value_places<DP>(0);
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) acc[i] = mfma32<DT>(value_frag<DP>(vt, at, k, i), pf[k], acc[i]);
    feed<2 * OB, 2>();
  }
  l = sum_halves(l);

  // the waves' parts join in LDS (behind their last reads of it); a wave then holds PER 32-column blocks
  constexpr int PER = OB / WK > 0 ? OB / WK : 1;
  float* const ml = (float*)(lds + WK * DP * 32 * 4);
  static_assert(WK * DP * 32 * 4 + WK * 65 * 4 <= G::LDS, "the parts fit the stages");
  barrier();
  if (h == 0) {
    ml[wave * 64 + q] = m;
    ml[wave * 64 + 32 + q] = l;
  }
  int* const strange_by = (int*)(ml + WK * 64);
  if (lane == 0) strange_by[wave] = strange;
  barrier();
  strange = false;
#pragma unroll
  for (int w = 0; w < WK; ++w) strange |= strange_by[w] != 0;
  float to = -INFINITY;
#pragma unroll
  for (int w = 0; w < WK; ++w) to = fmaxf(to, ml[w * 64 + q]);
  const float by = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
  l = 0.f;
#pragma unroll
  for (int w = 0; w < WK; ++w) {
    const float mw = ml[w * 64 + q];
    l += ml[w * 64 + 32 + q] * (mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - to));
  }
  float* const po = (float*)lds;
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) po[((wave * OB + i) * 16 + k) * 64 + lane] = acc[i][k] * by;
  barrier();
  const int i0 = wave * PER;
  if (!row.live || i0 >= OB) return;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) s += po[((w * OB + i0 + i) * 16 + k) * 64 + lane];
      acc[i][k] = s;
    }
  if (strange) {
    const Taken from = it.taken(32, 32 * WK);
#pragma unroll 1
    for (int key = from.first; key < min(limit, from.last); ++key)
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int d = 32 * (i0 + i) + 8 * k + 4 * h;
          if (d >= D) continue;
          const f32x4 v = strange_at<DT>(from, key, d);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][4 * k + e] += v[e];
        }
  }
  if (h == 0 && i0 == 0) write_stats<DT>(args, row.out, it.part, to, l);
  write_out<DT, DP, PER>(args, row.out, it.part, acc, 32 * i0, h, l);
}

// 128 rows, tiles of 64 keys in two stages of K and of V.
//
// Heads up to 128: four waves of 32 rows, two such workgroups a CU, whose turns
// cover each other's waits. One barrier a tile, behind the wait for its loads:
// by then every wave is done with the tile before, whose place the next one's
// loads take.
//
// Heads of 256 (PAIR): output and query of 32 rows are 192 registers, which
// would leave a SIMD one wave. Two waves share 32 rows, eight a workgroup, one a
// CU: each scores half of a tile's keys (all of D), they exchange their maxima
// and probabilities through LDS, and each sums half of the columns over all
// keys: two waves a SIMD, at the LDS traffic of the narrower heads. Both are in
// the same phase, so that the scores of tile j + 1 are formed beside the
// probabilities of tile j (the exponentials issue in the shadow of the
// products). One barrier a tile: behind it (probabilities of j and maxima of
// j + 1 written, V of j and K of j + 2 arrived) K of j + 1 and V of j - 1 are
// free for K of j + 3 and V of j + 1. A wave writes its exchange's places again
// only when the other has counted its turn, which it does behind its reads: a
// wait that finds the count there, since the writes come most of a tile later.
template <int DP>
struct Big {
  static constexpr bool PAIR = DP == 256;
  static constexpr int WAVES = PAIR ? 8 : 4, KT = 64, TILE = KT * DP * 2;
  static constexpr int SU = PAIR ? 1 : KT / 32, OB = PAIR ? 4 : DP / 32;  // score tiles and output blocks of a wave
  // places: K, K, V, V; the queries before the first V; then the exchange
  static constexpr int QUERY = 2 * TILE, QUERY_BYTES = kTileRows * DP * 2;
  static constexpr int PROBS = 4 * TILE, MAXIMA = PROBS + 8 * 2048;
  static constexpr int PLAIN = 4 * TILE > QUERY + QUERY_BYTES ? 4 * TILE : QUERY + QUERY_BYTES;
  static constexpr int TURNS = MAXIMA + 8 * 128, STRANGE = PAIR ? TURNS + 8 * 4 : PLAIN, LDS = STRANGE + 16;
  static_assert(WAVES * 8192 <= PLAIN, "the rows' way out fits");
};

template <int DT, int DP, bool STACKED, bool FULL>
__device__ __forceinline__ void sweep_big(const AttnArgs& args, uint8_t* lds, const Item& it) {
  using G = Big<DP>;
  using L = Loader<DP, G::KT, G::WAVES>;
  constexpr bool PAIR = G::PAIR;
  constexpr int KT = G::KT, SU = G::SU, OB = G::OB, STEPS = DP / 16;
  constexpr int KEYS32 = PAIR ? 2 : SU;  // 32s of keys of a tile
  constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
  const actune_prefix_attention_args& p = args.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rg = PAIR ? wave >> 1 : wave, hf = PAIR ? wave & 1 : 0, q = lane & 31, h = lane >> 5;
  const int D = FULL ? DP : (int)p.D;
  const L loader(D, wave, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds);
  const int n = it.na + it.nb;
  auto first_of = [&](int j) { return (j < it.na ? it.a0 + j : it.b0 + j - it.na) * KT; };
  auto key_tile = [&](int j) {
    const Keys& s = j < it.na ? it.pre : it.own;
    return L::tile(s.k, s.k_bytes, first_of(j), s.end, (j & 1) * G::TILE);
  };
  auto value_tile = [&](int j) {
    const Keys& s = j < it.na ? it.pre : it.own;
    return L::tile(s.v, s.v_bytes, first_of(j), s.end, (2 + (j & 1)) * G::TILE);
  };
  // whether key i of tile j exists and is not masked, in lane i (a load in flight where there is a mask)
  auto flag = [&](int j) -> uint32_t {
    const bool in_pre = j < it.na;
    const int key = first_of(j) + lane;
    uint32_t there = lane < KT && key < (in_pre ? it.pre.end : it.own.end);
    if (there && in_pre && it.pre.mask) there = it.pre.mask[key];
    return there;
  };
  uint64_t bits = 0, next_bits = 0;
  if (n > 0) {
    loader.request_keys(key_tile(0));
    if (PAIR && n > 1) loader.request_keys(key_tile(1));
  }
  loader.clear_columns(lds + wave * L::BLOCKS * 1024);
  loader.clear_columns(lds + G::TILE + wave * L::BLOCKS * 1024);
  const Row row = row_of<STACKED>(args, it.group_or_seq, it.head, it.row0 + 32 * rg + q, it.end);
  const bool busy = __any(row.live);  // (the same for both waves of a pair; the others only load)
  // queries by whole rows: a wave's (PAIR: its half of the pair's) rows to LDS
  u16x8 qf[STEPS];
  {
    constexpr int ROWS = PAIR ? 16 : 32, RPB = 512 / DP, QB = ROWS / RPB;
    const uint32_t at = __builtin_amdgcn_readfirstlane(loader.origin + G::QUERY + (32 * rg + 16 * hf) * DP * 2);
    const uint64_t from = (uint64_t)row.q;
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int r = 16 * hf + i * RPB + lane / (DP / 8);
      const uint32_t lo = __shfl((int)(uint32_t)from, r), hi = __shfl((int)(uint32_t)(from >> 32), r);
      uint32_t c = 16 * ((lane % (DP / 8)) ^ swizzle<DP>(r));
      c = c < (uint32_t)(2 * D) ? c : 0;
      dma16((const uint8_t*)(((uint64_t)hi << 32) | lo) + c, at + i * 1024);
    }
  }
  uint32_t there = 0;  // (solo) tile 1's
  if (n > 0) bits = __ballot(flag(0) != 0);
  if (n > 1) {
    if constexpr (PAIR) next_bits = __ballot(flag(1) != 0);
    else there = flag(1);
  }
  f32x16 acc[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
  float m = -INFINITY, l = 0.f;
  // the first own key that causal hides from this query
  const int limit = p.causal ? it.own.end - (int)p.T + row.t + 1 : INT_MAX;
  auto open_of = [&](int j) { return j < it.na ? INT_MAX : limit - first_of(j); };
  float* const maxima = (float*)(lds + G::MAXIMA);
  u16x8* const probs = (u16x8*)(lds + G::PROBS);
  volatile __attribute__((address_space(3))) int* const turns =
      (volatile __attribute__((address_space(3))) int*)(lds + G::TURNS);
  if (PAIR && lane == 0) turns[wave] = 0;
  volatile __attribute__((address_space(3))) int* const strange =
      (volatile __attribute__((address_space(3))) int*)(lds + G::STRANGE);
  if (threadIdx.x == 0) *strange = 0;

  f32x16 sc[SU];
  float top = -INFINITY;
  wait_loads();
  barrier();
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int r = 32 * rg + q;
    qf[s] = *(const u16x8*)(lds + G::QUERY + r * DP * 2 + 16 * ((2 * s + h) ^ swizzle<DP>(r)));
    if (D < DP && 16 * s + 8 * h >= D) qf[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
  barrier();
  if (n > 0) loader.request_values(value_tile(0));
  // scores of a tile without what stands beside them, masked, and their maximum
  auto score = [&](int j) {
#pragma unroll
    for (int u = 0; u < SU; ++u) sc[u] = score_tile<DT, DP>(lds + (j & 1) * G::TILE, 32 * (PAIR ? hf : u), qf);
    feed<SU * STEPS, 1>();
    settle(sc[0], sc[SU - 1]);
    mask_scores<KT>(sc, bits, open_of(j), hf, h);
    top = -INFINITY;
#pragma unroll
    for (int u = 0; u < SU; ++u) top = highest(sc[u], top);
    top = max_halves(top);
  };
  // raises the maximum for the tile in sc where it has to; what is subtracted from its scores
  auto settle_maximum = [&]() {
    top *= args.factor;
    if (__any(top > m + kLag)) {
      const float by = raise(m, top);
      l *= by;
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[i][k] *= by;
    }
    top = -INFINITY;
    return m == -INFINITY ? 0.f : m - lift<DT>();
  };
  // this wave's (and, PAIR, the other's) probabilities of a tile to where its values are summed
  auto hand_over = [&](const u16x8(&pf)[2 * SU], int turn) {
    // (the other wave's count of the turn before does not depend on anything that this one has yet to do)
    while (turns[wave ^ 1] < turn) __builtin_amdgcn_s_sleep(1);
    probs[(2 * wave) * 64 + lane] = pf[0];
    probs[(2 * wave + 1) * 64 + lane] = pf[1];
    if (h == 0) maxima[wave * 32 + q] = top;
  };
  auto sum_values = [&](const uint8_t* vt, const u16x8(&pf)[2 * SU]) {
    u16x8 pa[2 * KEYS32];
    if constexpr (PAIR) {
#pragma unroll
      for (int k = 0; k < 4; ++k) pa[k] = probs[(2 * (wave & ~1) + k) * 64 + lane];
      top = fmaxf(top, maxima[(wave ^ 1) * 32 + q]);
    } else {
#pragma unroll
      for (int k = 0; k < 2 * SU; ++k) pa[k] = pf[k];
    }
    const ValuePlace at = value_places<DP>(128 * hf);
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int k = 0; k < 2 * KEYS32; ++k) acc[i] = mfma32<DT>(value_frag<DP>(vt, at, k, i), pa[k], acc[i]);
    feed<2 * KEYS32 * OB, 2>();
  };
  auto clear_masked = [&](uint8_t* vt, int j) {
    const bool divided = j >= it.na && it.divides(first_of(j), KT);
    if (bits == kAll && !divided) return;
    if (bits != kAll) clear_rows<DP, KT>(vt, bits, (int)threadIdx.x, 64 * G::WAVES);
    if (divided && take_strange<DT, DP, KT>(vt, (int)threadIdx.x, 64 * G::WAVES)) *strange = 1;
    barrier();
  };

  if constexpr (PAIR) {
    if (n > 0 && busy) score(0);
    if (h == 0) maxima[wave * 32 + q] = top;
    barrier();
    top = fmaxf(top, maxima[(wave ^ 1) * 32 + q]);
    if (n > 2) loader.request_keys(key_tile(2));
    barrier();
    for (int j = 0; j + 1 < n; ++j) {
      const uint8_t* const kt = lds + ((j + 1) & 1) * G::TILE;
      uint8_t* const vt = lds + (2 + (j & 1)) * G::TILE;
      uint32_t there = 0;
      if (j + 2 < n) there = flag(j + 2);
      u16x8 pf[2 * SU];
      if (busy) {
        const float less = settle_maximum();
        f32x16 nx[SU];
        scores_beside<DT, DP, SU>(kt, 32 * hf, qf, nx, sc, args.factor, less, pf, l);
        settle(nx[0], nx[SU - 1]);
        mask_scores<KT>(nx, next_bits, open_of(j + 1), hf, h);
#pragma unroll
        for (int u = 0; u < SU; ++u) {
          top = highest(nx[u], top);
          sc[u] = nx[u];
        }
        top = max_halves(top);
      }
      if (busy) hand_over(pf, j);
      wait_loads();
      barrier();
      clear_masked(vt, j);
      const uint64_t ahead = __ballot(there != 0);
      loader.request_values(value_tile(j + 1));
      if (j + 3 < n) loader.request_keys(key_tile(j + 3));
      if (busy) sum_values(vt, pf);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (lane == 0) turns[wave] = j + 1;
      bits = next_bits;
      next_bits = ahead;
    }
    if (n > 0) {
      uint8_t* const vt = lds + (2 + ((n - 1) & 1)) * G::TILE;
      u16x8 pf[2 * SU];
      if (busy) {
        const float less = settle_maximum();
#pragma unroll
        for (int u = 0; u < SU; ++u) probabilities<DT>(sc[u], args.factor, less, pf + 2 * u, l);
      }
      if (busy) hand_over(pf, n - 1);
      wait_loads();
      barrier();
      clear_masked(vt, n - 1);
      if (busy) sum_values(vt, pf);
    }
  } else {
    for (int j = 0; j < n; ++j) {
      wait_loads();
      barrier();
      const uint64_t ahead = __ballot(there != 0);
      if (j + 1 < n) {
        if (j + 2 < n) there = flag(j + 2);
        loader.request_keys(key_tile(j + 1));
        loader.request_values(value_tile(j + 1));
      }
      uint8_t* const vt = lds + (2 + (j & 1)) * G::TILE;
      clear_masked(vt, j);
      if (busy && bits) {
        score(j);
        const float less = settle_maximum();
        u16x8 pf[2 * SU];
#pragma unroll
        for (int u = 0; u < SU; ++u) probabilities<DT>(sc[u], args.factor, less, pf + 2 * u, l);
        sum_values(vt, pf);
      }
      bits = ahead;
    }
  }
  barrier();  // the tiles are done with
  l = sum_halves(l);
  if constexpr (PAIR) {
    if (h == 0) maxima[wave * 32 + q] = l;
    barrier();
    l = maxima[(wave & ~1) * 32 + q] + maxima[(wave | 1) * 32 + q];
  }
  // the row is found again: its place costs the loop no registers
  int r = it.row0 + 32 * rg + q;
  asm volatile("" : "+v"(r));
  const Row end = row_of<STACKED>(args, it.group_or_seq, it.head, r, it.end);
  if (!busy) return;
  if (end.live && h == 0 && hf == 0) write_stats<DT>(args, end.out, it.part, m, l);
  const Taken from = it.taken(KT, KT);
  const int seen = !*strange ? 0 : p.causal ? it.own.end - (int)p.T + end.t + 1 : 0;  // keys that this row sees
  write_rows<DT, DP, OB>(args, lds + wave * 8192, end.live ? end.out : -1, it.part, acc, 128 * hf, l, from, seen);
}

// Workgroups go to the 8 XCDs in turn, each with its own L2: item order with
// an XCD's workgroups on consecutive items, which share their keys.
__device__ __forceinline__ int xcd_order(int id, int n) {
  const int x = id % kXcdCount, rest = n % kXcdCount;
  return x * (n / kXcdCount) + min(x, rest) + id / kXcdCount;
}

__device__ __forceinline__ Keys prefix_keys(const actune_prefix_attention_args& p, int g, int head) {
  const int most = (int)p.P;
  return Keys{(const uint16_t*)p.prefix_k + g * p.prefix_k_stride[0] + head * p.prefix_k_stride[2],
              (const uint16_t*)p.prefix_v + g * p.prefix_v_stride[0] + head * p.prefix_v_stride[2],
              (uint32_t)(p.prefix_k_stride[1] * 2), (uint32_t)(p.prefix_v_stride[1] * 2),
              p.prefix_mask ? p.prefix_mask + g * p.mask_stride : nullptr,
              p.prefix_lengths ? min(max(p.prefix_lengths[g], 0), most) : most};
}
__device__ __forceinline__ Keys own_keys(const actune_prefix_attention_args& p, int b, int head) {
  const int most = (int)p.S;
  return Keys{(const uint16_t*)p.k + b * p.k_stride[0] + head * p.k_stride[2],
              (const uint16_t*)p.v + b * p.v_stride[0] + head * p.v_stride[2], (uint32_t)(p.k_stride[1] * 2),
              (uint32_t)(p.v_stride[1] * 2), nullptr, p.lengths ? min(max(p.lengths[b], 0), most) : most};
}

constexpr int small_waves(int DP) { return DP == 256 ? 2 : 4; }
template <int DP, bool BIG>
struct Shape {
  static constexpr int WAVES = BIG ? Big<DP>::WAVES : small_waves(DP), ROWS = BIG ? kTileRows : kSmallRows;
  static constexpr int KEYS = BIG ? Big<DP>::KT : 32 * WAVES;  // of a tile
  static constexpr int LDS = BIG ? Big<DP>::LDS : Small<DP, small_waves(DP)>::LDS;
};

// Items in order: main items by group, key head, key split, (joint: sequence),
// row tile; then, stacked, the own keys' by sequence, head, split, row tile.
template <int DT, int DP, bool BIG, bool STACKED, bool FULL>
__global__ __launch_bounds__((64 * Shape<DP, BIG>::WAVES), BIG ? 2 : 1) void attend(const AttnArgs args) {
  extern __shared__ __align__(16) uint8_t attn_lds[];
  using S = Shape<DP, BIG>;
  const actune_prefix_attention_args& p = args.p;
  const int item = args.first + (int)blockIdx.x;
  const Keys none{nullptr, nullptr, 0, 0, nullptr, 0};
  Item it{none, none, 0, 0, 0, 0, 0, 0, 0, args.set_rows, 0, INT_MAX};
  if (!STACKED || item < args.main_items) {
    int id = xcd_order(item, args.main_items);
    it.row0 = take(id, args.tiles) * S::ROWS;
    const int seq = STACKED ? 0 : take(id, args.per_group_div);
    const int split = it.part = take(id, args.splits_div);
    it.head = take(id, args.heads);
    it.pre = prefix_keys(p, id, it.head);
    const int c0 = start_of(args.cut, split), c1 = start_of(args.cut, split + 1);
    it.a0 = min(c0, args.pre_cap);
    it.na = max(0, min(c1, (it.pre.end + S::KEYS - 1) / S::KEYS) - it.a0);
    it.group_or_seq = id;
    if constexpr (!STACKED) {
      it.group_or_seq = id * args.per_group + seq;
      it.own = own_keys(p, it.group_or_seq, it.head);
      // causal: keys past the last query of the tile are hidden from all of it
      const int last_t = min(quotient(it.row0 + S::ROWS - 1, args.share), (int)p.T - 1);
      if (p.causal) it.low = it.own.end - (int)p.T + quotient(it.row0, args.share) + 1;
      const int seen = p.causal ? min(it.own.end, it.own.end - (int)p.T + last_t + 1) : it.own.end;
      it.b0 = max(c0 - args.pre_cap, 0);
      it.nb = max(0, min(c1 - args.pre_cap, (max(seen, 0) + S::KEYS - 1) / S::KEYS) - it.b0);
    }
  } else {
    int id = item - args.main_items;
    const int tile = take(id, args.own_tiles) * S::ROWS;
    const int split = take(id, args.own_splits);
    it.part = args.splits + split;
    it.head = take(id, args.heads);
    it.own = own_keys(p, id, it.head);
    const int seq = take(id, args.per_group_div);
    it.group_or_seq = id;
    it.row0 = seq * args.seq_rows + tile;
    if (p.causal) it.low = it.own.end - (int)p.T + quotient(tile, args.share) + 1;
    it.end = (seq + 1) * args.seq_rows;
    it.b0 = start_of(args.own_cut, split);
    it.nb = max(0, min(start_of(args.own_cut, split + 1), (it.own.end + S::KEYS - 1) / S::KEYS) - it.b0);
  }
  if constexpr (BIG) sweep_big<DT, DP, STACKED, FULL>(args, attn_lds, it);
  else sweep_small<DT, DP, S::WAVES, STACKED, FULL>(args, attn_lds, it);
}

// Joins the parts of a row in one pass: DP / 4 lanes hold four columns each,
// groups of that many lanes take parts in turn, four in flight, with a maximum
// of their own, and then meet. W waves a row, which meet in LDS: as many as take
// most sets of parts in a round or two (128 rows of 256 in 256 parts: 25 us with
// four waves, 10.4 with sixteen; 768 rows of 128 in 14 parts: 5.0 us with one,
// 4.8 with four).
struct Joined {
  f32x4 o;
  float m, l;
  // with another's (neither's maximum is NaN)
  __device__ __forceinline__ void add(const f32x4& o2, float m2, float l2) {
    const float to = fmaxf(m, m2);
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
    const float b = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - to);
    l = m2 == -INFINITY ? l : m == -INFINITY ? l2 : a * l + b * l2;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = m2 == -INFINITY ? o[e] : m == -INFINITY ? o2[e] : fmaf(b, o2[e], a * o[e]);
    m = to;
  }
};
template <int DT, int DP, int W>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void join(const AttnArgs args) {
  constexpr int LANES = DP / 4, GROUPS = 64 / LANES * W;
  __shared__ float meet[W][6 * 64];
  const actune_prefix_attention_args& p = args.p;
  const int64_t rows = p.B * p.T * p.Hq, row = args.first + (int64_t)blockIdx.x * (W > 1 ? 1 : 4) + (W > 1 ? 0 : threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = 4 * (lane % LANES), D = (int)p.D;
  const int grp = (W > 1 ? wave * (64 / LANES) : 0) + lane / LANES;
  const float* const ml = args.part_ml + 2 * row;
  const float* const po = args.part_o + row * DP + min(col, D - 4);
  Joined sum{{0.f, 0.f, 0.f, 0.f}, -INFINITY, 0.f};
  for (int i0 = grp; i0 < args.parts; i0 += 4 * GROUPS) {
    float2 s[4];
    f32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = min(i0 + k * GROUPS, args.parts - 1);
      s[k] = *(const float2*)(ml + 2 * i * rows);
      v[k] = *(const f32x4*)(po + i * rows * DP);
    }
    // (a part without keys wrote no output worth reading: its maximum is -inf)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i0 + k * GROUPS < args.parts) sum.add(v[k], s[k].x, s[k].y);
  }
#pragma unroll
  for (int d = LANES; d < 64; d *= 2) {
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __shfl_xor(sum.o[e], d);
    sum.add(o, __shfl_xor(sum.m, d), __shfl_xor(sum.l, d));
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) meet[wave][64 * e + lane] = sum.o[e];
    meet[wave][256 + lane] = sum.m;
    meet[wave][320 + lane] = sum.l;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w)
      sum.add(f32x4{meet[w][lane], meet[w][64 + lane], meet[w][128 + lane], meet[w][192 + lane]}, meet[w][256 + lane],
              meet[w][320 + lane]);
  }
  if (lane >= LANES) return;
  const float l = sum.l;
  if (p.lse && lane == 0)
    p.lse[row] = l == 0.f ? -INFINITY : (sum.m - lift<DT>() + __builtin_log2f(l)) * 0.693147180559945309f;
  if (col >= D) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  u16x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = to16<DT>(sum.o[e] * inv);
  *(u16x4*)((uint16_t*)p.out + row * D + col) = v;
}

int padded(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

bool sizes_ok(const actune_prefix_attention_args& p) {
  if (p.B < 0 || p.T < 0 || p.G < 1 || p.Hkv < 1 || p.Hq < 1 || p.P < 0 || p.S < 0) return false;
  if (p.D < 8 || p.D > 256 || p.D % 8 || p.Hq % p.Hkv || p.B % p.G) return false;
  // rows and keys are counted in 32 bits, addresses in 64
  if (p.B > INT_MAX || p.T > INT_MAX || p.Hq > 1 << 20 || p.P > INT_MAX / 2 || p.S > INT_MAX / 2) return false;
  return p.B * p.T <= INT_MAX / 2 / p.Hq;
}

// What a workgroup of a shape costs beside its tiles of keys, and a tile, in us
// (measured alone and on a full chip: 128 rows of heads of 256 take 8.9 us with
// one tile and 14.8 with four, of 128 6.8 and 10.0; 32 rows 8.0 and 13.0, 5.8
// and 8.2 with tiles of 64 and 128 keys), and how many the chip holds at a time.
// Two workgroups a CU that are at work throughout slow each other: eight prompts
// of 512 with heads of 128 take 2.2 us a tile, 190 us where these give 134.
struct Cost {
  double fixed, tile;
  int slots;
};
Cost cost_of(int DP, bool big) {
  if (big) return DP == 256 ? Cost{7.0, 2.2, kCus} : DP == 128 ? Cost{5.7, 1.5, 2 * kCus} : Cost{4.3, 1.1, 4 * kCus};
  return DP == 256 ? Cost{6.3, 1.7, kCus} : DP == 128 ? Cost{4.9, 0.9, kCus} : Cost{3.8, 0.7, 2 * kCus};
}

struct Sizes {
  int64_t rows, per, out_rows;  // rows of a sequence and key head; sequences of a group; rows of the output
  int DP;
};

// The cheapest cut of a way to lay out the rows, and its time in us.
double cut_plan(const actune_prefix_attention_args& p, const Sizes& z, bool big, bool stacked, Plan& g) {
  auto tiles = [](int64_t n, int64_t tr) { return (n + tr - 1) / tr; };
  const Cost c = cost_of(z.DP, big);
  const int64_t tr = big ? kTileRows : kSmallRows, tk = big ? 64 : 32 * small_waves(z.DP);
  g = Plan{};
  g.big = big;
  g.stacked = stacked;
  g.tiles = (int)tiles(stacked ? z.rows * z.per : z.rows, tr);
  g.pre_cap = tiles(p.P, tk);
  g.own_cap = tiles(p.S, tk);
  const int64_t sets = (stacked ? p.G : p.B) * p.Hkv * g.tiles, cap = g.pre_cap + (stacked ? 0 : g.own_cap);
  int64_t own = 0;
  if (stacked && p.S > 0) {
    g.own_tiles = (int)tiles(z.rows, tr);
    own = p.B * p.Hkv * g.own_tiles;
    // own keys: an item as long as a few of the main items' tiles; they fill what the chip has left, before the main
    // items are cut for the rest
    const int64_t want = own >= c.slots ? 1 : (c.slots + own - 1) / own, most = (g.own_cap + 3) / 4;
    g.own_splits = (int)(want < most ? want : most);
    if (g.own_splits < 1) g.own_splits = 1;
  }
  g.own_items = own * g.own_splits;
  const int64_t own_len = own ? tiles(g.own_cap, g.own_splits) : 0;
  double best = -1;
  for (int k = 0; k <= 4; ++k) {
    int64_t s = k == 0 ? 1 : (k * c.slots - (k == 1 ? g.own_items % c.slots : 0)) / sets;
    s = s < 1 ? 1 : s;
    s = s > cap ? cap : s;
    if (s < 1) s = 1;
    const int64_t items = sets * s, len = tiles(cap, s), parts = s + (own ? g.own_splits : 0);
    const double main_time = c.fixed + c.tile * len, own_time = c.fixed + c.tile * own_len;
    double t;
    if (items + g.own_items <= c.slots) t = main_time > own_time ? main_time : own_time;
    else if (!own) t = (double)tiles(items, c.slots) * main_time;
    else t = 1.1 * (items * main_time + g.own_items * own_time) / c.slots + 0.5 * main_time;
    // the join: a launch, and each part written and read once at about 4.5 TB/s
    if (parts > 1) t += 4.0 + (double)z.out_rows * parts * z.DP * 8 / 4.5e6;
    if (best < 0 || t < best) {
      best = t;
      g.splits = (int)s;
      g.main_items = items;
      g.parts = (int)parts;
    }
  }
  return best;
}

// The row layout, the tile height and the cut with the least estimated time.
// Each is the fastest somewhere (us, join included; rows of 32 / 128 and joint /
// stacked, best cut of each that was tried):
//                                          32 joint  32 stacked  128 joint  128 stacked
//   one chunk of 50, 8 heads of 256            15.8          -        16.5          -
//   32 chunks of 50, 8 heads of 256            70          91         40.7         48
//   24 tokens, 32 heads of 128, 4096 keys     106          42        168           38
//   48 tokens, 8 heads of 256, 65537 keys       -         109        357           53
//   8 prompts of 512, 32 heads of 128         381           -        190          260
// Cuts of the first: 18.9 with 4, 15.8 with 8, 16.6 with 14; of the second, one
// part 44 and two 40.7; of the fourth 77 with 34, 53 with 69, 61 with 85 (with
// 53, which the own keys' two splits leave: 61).
// 32-bit counts hold for every size that sizes_ok takes: items are at most rows
// plus a bounded number of splits of them.
Plan plan_of(const actune_prefix_attention_args& p) {
  const Sizes z{p.T * (p.Hq / p.Hkv), p.B / p.G, p.B * p.T * p.Hq, padded(p.D)};
  Plan best{}, g;
  double least = -1;
  for (int way = 0; way < 4; ++way) {
    const bool big = way & 1, stacked = way & 2;
    if (stacked && (z.per < 2 || p.P == 0)) continue;
    const double t = cut_plan(p, z, big, stacked, g);
    if (least < 0 || t < least) {
      least = t;
      best = g;
    }
  }
  return best;
}

int64_t part_rows(const actune_prefix_attention_args& p) { return p.B * p.T * p.Hq; }
int64_t ml_bytes(const actune_prefix_attention_args& p, const Plan& g) {
  return (g.parts * part_rows(p) * 8 + 255) / 256 * 256;
}
int64_t need_bytes(const actune_prefix_attention_args& p, const Plan& g) {
  return g.parts == 1 ? 0 : ml_bytes(p, g) + g.parts * part_rows(p) * padded(p.D) * 4;
}

// Items or rows of a launch: a dispatch holds less than 2^32 threads.
constexpr int64_t kMost = 1 << 21;

template <int DT, int DP, bool BIG, bool STACKED, bool FULL>
void launch_attend(AttnArgs a, int64_t items, hipStream_t st) {
  using S = Shape<DP, BIG>;
  if constexpr (S::LDS > 64 * 1024) allow_dynamic_lds<attend<DT, DP, BIG, STACKED, FULL>>(160 * 1024);
  constexpr int threads = 64 * S::WAVES, lds = S::LDS;
  for (int64_t first = 0; first < items; first += kMost) {
    a.first = (int)first;
    const int64_t n = items - first < kMost ? items - first : kMost;
    attend<DT, DP, BIG, STACKED, FULL><<<dim3((unsigned)n), threads, lds, st>>>(a);
  }
}

template <int DT, int DP, int W>
void launch_join(AttnArgs a, int64_t rows, hipStream_t st) {
  constexpr int each = W > 1 ? 1 : 4;  // rows of a workgroup
  for (int64_t first = 0; first < rows; first += kMost * each) {
    a.first = (int)first;
    const int64_t left = (rows - first + each - 1) / each, n = left < kMost ? left : kMost;
    join<DT, DP, W><<<dim3((unsigned)n), W > 4 ? 64 * W : 256, 0, st>>>(a);
  }
}

template <int DT, int DP, bool FULL>
void launch_sweep(const AttnArgs& a, const Plan& g, hipStream_t st) {
  const int64_t grid = g.main_items + g.own_items;
  if (g.big) {
    if (g.stacked) launch_attend<DT, DP, true, true, FULL>(a, grid, st);
    else launch_attend<DT, DP, true, false, FULL>(a, grid, st);
  } else {
    if (g.stacked) launch_attend<DT, DP, false, true, FULL>(a, grid, st);
    else launch_attend<DT, DP, false, false, FULL>(a, grid, st);
  }
}

template <int DT, int DP>
void launch(const AttnArgs& a, const Plan& g, hipStream_t st) {
  // Heads that fill the padded size load their keys without a choice of lanes (one chunk of 50, 8 heads of 256, 816
  // keys: 15.4 us for 16.3; 48 requests over 65537 keys: 61.5 for 64).
  if (a.p.D == DP) launch_sweep<DT, DP, true>(a, g, st);
  else launch_sweep<DT, DP, false>(a, g, st);
  const int64_t rows = part_rows(a.p);
  constexpr int ROUND = 4 * 64 / (DP / 4);  // parts that a wave has in flight
  if (g.parts > 8 * ROUND) launch_join<DT, DP, 16>(a, rows, st);
  else if (g.parts > ROUND) launch_join<DT, DP, 4>(a, rows, st);
  else if (g.parts > 1) launch_join<DT, DP, 1>(a, rows, st);
}

template <int DT>
void launch(const AttnArgs& a, const Plan& g, hipStream_t st) {
  const int DP = padded(a.p.D);
  if (DP == 64) launch<DT, 64>(a, g, st);
  else if (DP == 128) launch<DT, 128>(a, g, st);
  else launch<DT, 256>(a, g, st);
}

}  // namespace
}  // namespace actune

using namespace actune;

extern "C" {

int64_t actune_prefix_attention_workspace_bytes(const actune_prefix_attention_args* args) {
  if (!args || !sizes_ok(*args)) return -1;
  if (part_rows(*args) == 0) return 0;
  return need_bytes(*args, plan_of(*args));
}

int actune_prefix_attention(const actune_prefix_attention_args* args, void* stream) {
  block_clear_error();
  if (!args) return block_fail("null pointer");
  const actune_prefix_attention_args& p = *args;
  if (p.dtype != kBF16 && p.dtype != kF16) return block_fail("attention takes bf16 or f16");
  if (p.D < 8 || p.D > 256 || p.D % 8) return block_fail("head size must be a multiple of 8 up to 256");
  if (p.Hq < 1 || p.Hkv < 1 || p.Hq % p.Hkv) return block_fail("query heads must be a multiple of key heads");
  if (p.G < 1 || p.B < 0 || p.B % p.G) return block_fail("the batch must be whole groups, one for each prefix");
  if (!sizes_ok(p)) return block_fail("invalid dimensions");
  if (!(p.scale > 0.f) || !std::isfinite(p.scale)) return block_fail("scale must be finite and above zero");
  if (part_rows(p) == 0) return kOk;
  if (!p.q || !p.out || (p.P > 0 && (!p.prefix_k || !p.prefix_v)) || (p.S > 0 && (!p.k || !p.v)))
    return block_fail("null pointer");
  const int64_t most = (int64_t)1 << 40;
  for (int i = 0; i < 3; ++i) {
    const bool token = i == 1;
    for (int64_t s : {p.prefix_k_stride[i], p.prefix_v_stride[i], p.k_stride[i], p.v_stride[i]})
      if (s < 0 || s % 8 || s >= (token ? (int64_t)1 << 23 : most)) return block_fail("invalid stride of keys or values");
    if (p.q_stride[i] < 0 || p.q_stride[i] % 8 || p.q_stride[i] >= most) return block_fail("invalid stride of q");
  }
  if (p.mask_stride < 0 || p.mask_stride >= most) return block_fail("invalid mask stride");
  for (const void* t : {p.q, p.prefix_k, p.prefix_v, p.k, p.v, (const void*)p.out, (const void*)p.workspace})
    if (!is_aligned(t, 16)) return block_fail("misaligned operand (16 B)");
  if (!is_aligned(p.prefix_lengths, 4) || !is_aligned(p.lengths, 4) || !is_aligned(p.lse, 4))
    return block_fail("misaligned operand");
  const Plan g = plan_of(p);
  const int64_t need = need_bytes(p, g);
  if (need > 0 && (!p.workspace || p.workspace_bytes < need)) return block_fail("workspace too small");
  if (g.main_items + g.own_items > INT_MAX) return block_fail("invalid dimensions");
  AttnArgs a{};
  a.p = p;
  a.parts = g.parts;
  a.splits = g.splits;
  a.main_items = (int)g.main_items;
  a.pre_cap = (int)g.pre_cap;
  a.per_group = (int)(p.B / p.G);
  a.share = div_of(p.Hq / p.Hkv);
  a.seq_rows = (int)(p.T * (p.Hq / p.Hkv));
  a.set_rows = g.stacked ? a.seq_rows * a.per_group : a.seq_rows;
  a.rows = div_of(a.seq_rows);
  a.tiles = div_of(g.tiles);
  a.per_group_div = div_of(a.per_group);
  a.splits_div = div_of(g.splits);
  a.heads = div_of(p.Hkv);
  a.own_tiles = div_of(g.own_tiles > 0 ? g.own_tiles : 1);
  a.own_splits = div_of(g.own_splits > 0 ? g.own_splits : 1);
  a.cut = cut_of(g.pre_cap + (g.stacked ? 0 : g.own_cap), g.splits);
  a.own_cut = cut_of(g.own_cap, g.own_splits > 0 ? g.own_splits : 1);
  a.factor = p.scale * 1.44269504088896340736f;
  a.part_ml = (float*)p.workspace;
  a.part_o = (float*)((uint8_t*)p.workspace + (need > 0 ? ml_bytes(p, g) : 0));
  if (p.dtype == kBF16) launch<kBF16>(a, g, (hipStream_t)stream);
  else launch<kF16>(a, g, (hipStream_t)stream);
  return block_status();
}

}  // extern "C"
