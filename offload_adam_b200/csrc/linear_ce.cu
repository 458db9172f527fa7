// Softmax cross entropy of h W^T against labels, in pieces of the vocabulary, without the logits.
//
//   z_ij = sum_k h_ik W_jk        lse_i = log sum_j exp z_ij        loss_i = lse_i - z_i,label
//   d_ij = (exp(z_ij - lse_i) - [j = label_i]) g_i      dh = d W      dW = d^T h
//
// Rows whose label is ignored take no part: the others are packed first, so their work is saved
// and nothing that stands in them (a padded batch's NaN) reaches a sum.
//
// Precision.  A confident row's loss is the small difference of two large numbers, so it is not
// formed as one: packing computes the label's logit apart, in fp32 on the ordinary cores; the products'
// statistics leave that word out; and with their m and s
//     loss_i = log(1 + s exp(m - z_label)),    1 - p_label = 1 - exp(-loss_i)
// in fp64.  The gradient of the logits is held apart from its size: with q_i = 1 - p_label,
//     d_ij = q_i g_i (exp(z_ij - m_i) / s_i - [j = label_i]),    over the other words, as above
// so the label's entry, which most of a row's gradient hangs on, is -1 exactly in bf16; q_i g_i is
// applied to the fp32 sums of dh, and to the rows of h that go into dW (bf16, rounded once more).
// m and log s stay two numbers: their sum would lose the latter beside logits of 1e6, or of a mask's
// lowest value, and each word of such a row would have the whole of it.
// tcgen05 cuts off what it adds to an accumulator, towards zero each time: sums of terms of one sign
// lose 0.4e-7 to 1e-7 of their value with each addition of 16 terms.  Logits of 4096 terms came out 1e-5
// too small, the losses of unsure rows 2.5e-5 off, so the statistics take their logits in chains of 32
// additions (512 terms; 256 for few rows) that the epilogue adds up.  The logits that backward forms
// again come in chains of 8192 terms (of 2^18 terms in one chain, a logit of 32 was 0.05 off).  dW over
// 2^20 rows was 0.7 % too small, over 2^22 2.3 %, so an accumulator of the gradients takes kLceSumTerms
// of them, 4e-4 at most: dW of more rows is summed in fp32 in memory, a launch for every kLceSumTerms
// rows, and dh of more words in splits (in chains for few rows).
//
// Forward: one product whose epilogue keeps, per row and 128 words, the maximum and the sum of
// exponentials (8 bytes for 256 bytes of bf16 logits), and a small kernel that joins them (of a few
// rows the last block of the product).
// Backward, for each piece of the vocabulary: the product again, whose epilogue writes the
// gradient of the piece's logits in bf16, and one launch for both products that read it; dh is
// summed over the pieces in fp32 and rounded once.
//
// What bounds it: the products, at the rate of the library's (4096 rows, hidden 4096, 128256 words on
// a B200: forward 3.1 ms, 1.37 PFLOP/s, a bf16 product of the library's with nothing behind it 3.1;
// all 12.5 to 13.8 ms, four products, as the chip's power allows).  Small heads are bound by the
// exponentials (16 a cycle and SM), few rows by reading W (6.6 TB/s), the smallest calls by the host.
//
// All three products are one pipeline: a CTA pair computes a 256 x 256 tile with tcgen05 (each CTA
// 128 rows, half of B each), TMA fills six stages of 64 inner values, two accumulators in tensor
// memory let the epilogue of a tile overlap the products of the next, one pair per two SMs
// takes tiles in turn.
#include <cudaTypedefs.h>

#include <atomic>

#include "common.cuh"
#include "linear_ce.h"
#include "umma.cuh"

namespace oab {
namespace {

using namespace umma;

constexpr int kTile = kLceTile;
constexpr int kInner = 64;                              // inner values of a stage: 128 bytes
constexpr int kStages = 6;
constexpr int kHalfBytes = 128 * kInner * 2;            // one CTA's part of an operand's stage
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kEpilogueWarps = 16;       // eight for each accumulator
constexpr int kStagingBytes = 32 * 64;   // of an epilogue warp: 32 lines of 64 bytes on their way out
constexpr int smem_of(bool staging) { return kStages * kStageBytes + (staging ? kEpilogueWarps * kStagingBytes : 0) + 1024; }  // starts on 1024 bytes
constexpr int kGemmThreads = 64 + 32 * kEpilogueWarps;
constexpr int kChain = 8, kGradChain = 128;  // stages of a chain of the statistics, of the logits for backward
constexpr int kGroup = 16;  // row tiles that share a column tile in turn: 4096 rows of h stay in L2

enum Pass { kStats = 0, kLogitGrad = 1, kGrads = 2 };

struct GemmParams {
  CUtensorMap a, b;    // kStats, kLogitGrad: packed rows and W.  kGrads: d and W, for dh
  CUtensorMap a2, b2;  // kGrads: d and packed rows, for dW
  CUtensorMap out;     // kLogitGrad: d.  kGrads: dW, or with wacc its fp32 sums
  CUtensorMap out_acc; // kGrads: the fp32 sums of dh, by split
  const int* count;
  int64_t rows;        // capacity of the per-row arrays
  int64_t padded;
  int hidden;
  int64_t word0;       // first word of the piece
  int words;           // and how many
  int64_t* report;
  int* lost;           // set by a launch that gave up a wait: the results of all that follows are NaN
  uint64_t wait_limit;
  const int* label;
  // kStats
  float2* part;
  // kLogitGrad
  const float *top, *rest;
  const float *miss, *row_g;  // the latter by row, or null
  const int* index;
  const uint16_t* packed;
  int64_t row_pitch;          // of packed and scaled
  uint16_t* scaled;           // null: not wanted (again)
  uint16_t* gh;               // kLogitGrad: its ignored rows become zero; kGrads: dh goes out; null: neither
  const int64_t* labels;
  int64_t ignore;
  uint16_t* d;                // few rows; otherwise by `out`
  int64_t pitch;
  // kGrads
  const float *inv, *g;  // each may be null (1)
  int want_dh, want_dw;
  uint16_t* gw;               // few rows; otherwise by `out`
  int row0;                   // first packed row of the sums of dW
  int wacc;                   // dW goes to fp32 sums; those of row0 = 0 start them
  int splits;
  int first;             // piece: its dh starts the sums
};

// exp_of is off by about (|x| + 4) 2^-24 of its value
__device__ __forceinline__ float exp2_of(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float x) { return exp2_of(__fmul_rn(x, kLog2E)); }
// the softmax of a logit over the words that are not the label; `rest` in base 2
__device__ __forceinline__ float share_of(float z, float top, float rest) { return exp2_of(__fmaf_rn(__fsub_rn(z, top), kLog2E, -rest)); }
__device__ __forceinline__ float finite_shift(float m) { return m == -INFINITY ? 0.f : m; }

struct Tile {
  int kind;       // kGrads: 0 dh, 1 dW
  int m, n;       // first row and column
  int k0, steps;  // first inner value, stages
  int split;
  // kGrads: at most 128 hidden columns, so products of 128 columns (2000 rows of 64, 5000 words: 18.0 us
  // for 19.6; 622 rows of 840, 32003 words, a fourth of the tiles: 72.3 for 73.4)
  bool narrow;
};

// Tiles of a pass, and which of them a CTA pair takes.  Column tiles turn slower than up to kGroup
// row tiles.
struct Plan {
  int mt, nt, per_split, dh_tiles, wt, ht, total, k_steps, row_steps;
  int pairs, alone, first_dw;  // see pick
  template <int PASS>
  __device__ __forceinline__ void make(const GemmParams& p, int n_rows, int n_pairs) {
    mt = (n_rows + kTile - 1) / kTile;
    pairs = n_pairs;
    if (PASS == kGrads) {
      ht = (p.hidden + kTile - 1) / kTile;
      nt = ht;
      wt = p.want_dw ? (p.words + kTile - 1) / kTile : 0;
      per_split = mt * nt;
      dh_tiles = p.want_dh ? per_split * p.splits : 0;
      total = dh_tiles + wt * ht;
      k_steps = (p.words + kInner - 1) / kInner;
      const int left = n_rows - p.row0, own = left < 0 ? 0 : left < kLceSumTerms ? left : kLceSumTerms;
      row_steps = (own + kInner - 1) / kInner;
      // The tiles of dh are long (a sum over the words) and come first, those of dW (a sum over the
      // rows) fill up.  Pairs that a last, partial round of dh leaves idle take as many tiles
      // of dW as such a tile is long before the others join in.  4096 rows, hidden 4096, 32768
      // words: 256 tiles of dh for 74 pairs, 1481 us; shared out in turn 1575.
      alone = dh_tiles % pairs;
      first_dw = 0;
      if (alone != 0 && wt > 0) {
        // in stages; a tile of dW takes as long as its way out, about 7 stages, at least
        const int length = (k_steps + p.splits - 1) / p.splits, one = row_steps < 7 ? 7 : row_steps;
        const int64_t fill = (int64_t)(length / one) * (pairs - alone);
        first_dw = (int)(fill < (int64_t)wt * ht ? fill : (int64_t)wt * ht);
      }
    } else {
      nt = (p.words + kTile - 1) / kTile;
      total = mt * nt;
      k_steps = (p.hidden + kInner - 1) / kInner;
    }
  }
  // The `turn`-th tile of `pair`, or -1.
  template <int PASS>
  __device__ __forceinline__ int pick(int pair, int turn) const {
    if (PASS != kGrads) {
      const int t = pair + turn * pairs;
      return t < total ? t : -1;
    }
    const int rounds = dh_tiles / pairs + (pair < alone ? 1 : 0);
    if (turn < rounds) return pair + turn * pairs;
    turn -= rounds;
    if (pair >= alone && first_dw > 0) {
      const int idle = pairs - alone, own = first_dw / idle + (pair - alone < first_dw % idle ? 1 : 0);
      if (turn < own) return dh_tiles + (pair - alone) + turn * idle;
      turn -= own;
    }
    const int64_t t = (int64_t)dh_tiles + first_dw + pair + (int64_t)turn * pairs;
    return t < total ? (int)t : -1;
  }
  __device__ __forceinline__ static void place(int t, int mt, int nt, int& m, int& n) {
    const int g = t / (kGroup * nt), first = g * kGroup, r = t - g * kGroup * nt;
    const int gm = mt - first < kGroup ? mt - first : kGroup;
    m = first + r % gm;
    n = r / gm;
  }
  template <int PASS>
  __device__ __forceinline__ Tile at(const GemmParams& p, int t) const {
    Tile x;
    x.kind = 0;
    x.split = 0;
    x.k0 = 0;
    int m, n;
    if (PASS == kGrads) {
      if (t < dh_tiles) {
        x.split = t / per_split;
        place(t - x.split * per_split, mt, nt, m, n);
        const int lo = (int)((int64_t)k_steps * x.split / p.splits), hi = (int)((int64_t)k_steps * (x.split + 1) / p.splits);
        x.k0 = lo * kInner;
        x.steps = hi - lo;
      } else {
        x.kind = 1;
        x.k0 = p.row0;
        place(t - dh_tiles, wt, ht, m, n);
        x.steps = row_steps;
      }
    } else {
      place(t, mt, nt, m, n);
      x.steps = k_steps;
    }
    x.m = m * kTile;
    x.n = n * kTile;
    x.narrow = PASS == kGrads && p.hidden - x.n <= kTile / 2;
    return x;
  }
};

// ------------------------------------------------------------------- epilogues
// Of the gradients: every epilogue warp handles 32 rows (lanes) and 128 columns of the CTA's 128 x 256
// tile, and every other tile of its pair.  A warp is a chain of latencies (the accumulator is
// done, its load, a fence, the way out), so there are eight for each accumulator, and the accumulator
// is given back (`release`) with the last load from it, before anything is computed from that.
// Of the statistics likewise.  Where the sums of these or of the logits' gradient come in several chains,
// all sixteen take 64 columns of every tile.  (4096 rows of 128, 32000 words: 55 us by halves, 78 all together.)

struct RowValues {  // of the packed row that a thread has in a tile
  int label;
  float top, rest;
};
template <int PASS>
__device__ __forceinline__ RowValues row_values(const GemmParams& p, int row, int n_rows) {
  RowValues r{-1, 0.f, INFINITY};
  if (PASS != kGrads && row < n_rows) {
    r.label = p.label[row];
    if (PASS == kLogitGrad) {
      r.top = p.top[row];
      r.rest = p.rest[row];
    }
  }
  return r;
}

// {max, sum of exponentials} of a row's 64 logits from column `col` on, without the label's.
__device__ __forceinline__ float2 stats_of(float (&v)[64], int col, int words, int label) {
  const int left = words - col, hit = label - col;
  if (left < 64 || (hit >= 0 && hit < 64)) {
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (i >= left || i == hit) v[i] = -INFINITY;
  }
  float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 4; i < 64; ++i) top[i & 3] = fmaxf(top[i & 3], v[i]);
  const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), sh = finite_shift(m);
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 64; ++i) t[i & 3] = __fadd_rn(t[i & 3], exp_of(__fsub_rn(v[i], sh)));
  return make_float2(m, __fadd_rn(__fadd_rn(t[0], t[1]), __fadd_rn(t[2], t[3])));
}
__device__ __forceinline__ float2 join2(const float2& a, const float2& b) {
  const float m = fmaxf(a.x, b.x), sh = finite_shift(m);
  return make_float2(m, __fadd_rn(__fmul_rn(a.y, exp_of(__fsub_rn(a.x, sh))), __fmul_rn(b.y, exp_of(__fsub_rn(b.x, sh)))));
}

// A warp's 32 lines of 64 bytes leave through its staging buffer, 16-byte parts swizzled as TMA
// expects them (part c of line r at c ^ (r / 2 % 4), which also keeps the stores free of bank
// conflicts).  A store a thread, straight from its row, touched 32 lines an instruction.
__device__ __forceinline__ void stage_begin(int lane) {
  if (lane == 0) store_wait_read();
  __syncwarp();
}
__device__ __forceinline__ void stage_part(uint32_t staging, int lane, int c, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  st_shared16(staging + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4), w0, w1, w2, w3);
}
// 32 columns as bf16
__device__ __forceinline__ void stage_bf16(uint32_t staging, int lane, const float (&v)[32]) {
  stage_begin(lane);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    stage_part(staging, lane, c, f32x2_to_bf16x2_rne(v[8 * c], v[8 * c + 1]), f32x2_to_bf16x2_rne(v[8 * c + 2], v[8 * c + 3]),
               f32x2_to_bf16x2_rne(v[8 * c + 4], v[8 * c + 5]), f32x2_to_bf16x2_rne(v[8 * c + 6], v[8 * c + 7]));
  store_fence();
  __syncwarp();
}

// What the epilogue warps of the gradient of the logits do while the first products run, the
// `mine`-th of `all` warps: scaled[k] = packed[k] (1 - p_label) g, the rows of h as dW takes them,
// rounded to bf16 and padded with zeros likewise; and the zero rows of gh.
__device__ __forceinline__ void prepare_rows(const GemmParams& p, int n_rows, int mine, int all) {
  const int vecs = p.hidden >> 3, lane = threadIdx.x & 31;
  if (p.gh != nullptr) {
    for (int64_t r = mine; r < p.rows; r += all) {
      if (p.labels[r] != p.ignore) continue;
      uint4* to = reinterpret_cast<uint4*>(p.gh + r * p.hidden);
      for (int v = lane; v < vecs; v += 32) to[v] = make_uint4(0, 0, 0, 0);
    }
  }
  if (p.scaled == nullptr) return;
  for (int k = mine; k < (n_rows + kLceRowPad - 1) / kLceRowPad * kLceRowPad; k += all) {
    float c = k < n_rows ? p.miss[k] : 0.f;
    if (k < n_rows && p.row_g != nullptr) c = __fmul_rn(c, p.row_g[p.index[k]]);
    const uint4* from = reinterpret_cast<const uint4*>(p.packed + (int64_t)k * p.row_pitch);  // zeros beyond n_rows
    uint4* to = reinterpret_cast<uint4*>(p.scaled + (int64_t)k * p.row_pitch);
    auto both = [c](uint32_t w) {
      return f32x2_to_bf16x2_rne(__fmul_rn(__uint_as_float(w << 16), c), __fmul_rn(__uint_as_float(w & 0xffff0000u), c));
    };
#pragma unroll 4
    for (int v = lane; v < vecs; v += 32) {
      const uint4 f = from[v];
      to[v] = make_uint4(both(f.x), both(f.y), both(f.z), both(f.w));
    }
  }
}

// 32 of a row's logits become their gradient, and go out.
__device__ __forceinline__ void logit_grad_part(const GemmParams& p, float (&v)[32], int col, int row, uint32_t staging, int lane,
                                                const RowValues& values, bool counts) {
  const int lab = values.label >= 0 ? (int)(values.label - p.word0) : -1;
  const float top = values.top, rest = values.rest;
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = share_of(v[i], top, rest);
  const int hit = lab - col;
  if (lab >= 0 && hit >= 0 && hit < 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i == hit) v[i] = -1.f;
  }
  // the zero rows behind the last one, which pad the inner dimension of dW: where a word of W holds an
  // infinity their logits are NaN
  if (!counts) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.f;
  }
  stage_bf16(staging, lane, v);
  if (lane == 0) {
    if (col < p.words && row < p.padded) tma_store(&p.out, staging, col, row);
    store_commit();
  }
}

template <class Release>
__device__ __forceinline__ void logit_grad_tile(const GemmParams& p, const Tile& x, uint32_t tmem, int row, int half, uint32_t staging,
                                                int lane, const RowValues& values, bool counts, const Release& release) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float v[32];
    tmem_load32(tmem + c * 32, v);
    if (c == 3) release();
    logit_grad_part(p, v, x.n + half * 128 + c * 32, row, staging, lane, values, counts);
  }
}

__device__ __forceinline__ void store_bf16x8(uint16_t* at, const float* v, float scale) {
  uint4 o;
  o.x = f32x2_to_bf16x2_rne(__fmul_rn(v[0], scale), __fmul_rn(v[1], scale));
  o.y = f32x2_to_bf16x2_rne(__fmul_rn(v[2], scale), __fmul_rn(v[3], scale));
  o.z = f32x2_to_bf16x2_rne(__fmul_rn(v[4], scale), __fmul_rn(v[5], scale));
  o.w = f32x2_to_bf16x2_rne(__fmul_rn(v[6], scale), __fmul_rn(v[7], scale));
  *reinterpret_cast<uint4*>(at) = o;
}
// What all rows of dh, and dW, are multiplied by.
__device__ __forceinline__ float all_scale(const float* inv, const float* g, const int* lost) {
  float scale = *lost != 0 ? NAN : 1.f;
  if (inv != nullptr) scale = __fmul_rn(scale, *inv);
  return g != nullptr ? __fmul_rn(scale, *g) : scale;
}
__device__ __forceinline__ float all_scale(const GemmParams& p) { return all_scale(p.inv, p.g, p.lost); }
// What packed row k of dh is multiplied by, beside the scale of all rows.
__device__ __forceinline__ float row_scale(const GemmParams& p, int k, float scale) {
  scale = __fmul_rn(scale, p.miss[k]);
  return p.row_g != nullptr ? __fmul_rn(scale, p.row_g[p.index[k]]) : scale;
}

// 16 columns as fp32 on their way to sums in memory.
__device__ __forceinline__ void stage_sums(uint32_t staging, int lane, const Tile& x, float (&v)[16]) {
  if (x.steps == 0) {  // nothing was summed
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.f;
  }
  stage_begin(lane);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    stage_part(staging, lane, i, __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
               __float_as_uint(v[4 * i + 3]));
  store_fence();
  __syncwarp();
}

template <class Release>
__device__ __forceinline__ void dh_tile(const GemmParams& p, const Tile& x, uint32_t tmem, int row, int n_rows, int half, float scale,
                                        uint32_t staging, int lane, const Release& release) {
  uint16_t* out = nullptr;
  if (p.gh != nullptr && row < n_rows) {  // one piece, one split: these are the whole sums
    out = p.gh + (int64_t)p.index[row] * p.hidden;
    scale = row_scale(p, row, scale);
  }
#pragma unroll 1
  for (int c = 0; c < 8; ++c) {
    float v[16];
    tmem_load16(tmem + c * 16, v);
    if (c == 7) release();
    const int col = x.n + half * 128 + c * 16;
    if (p.gh != nullptr) {
      if (out != nullptr && col < p.hidden) store_bf16x8(out + col, v, scale);
      if (out != nullptr && col + 8 < p.hidden) store_bf16x8(out + col + 8, v + 8, scale);
      continue;
    }
    stage_sums(staging, lane, x, v);  // no stage: a last piece of fewer stages than splits
    if (lane == 0) {
      if (col < p.hidden && row < n_rows) tma_store3(&p.out_acc, staging, col, row, x.split, !p.first);
      store_commit();
    }
  }
}

template <class Release>
__device__ __forceinline__ void dw_tile(const GemmParams& p, const Tile& x, uint32_t tmem, int row, int half, float scale,
                                        uint32_t staging, int lane, const Release& release) {
  if (p.wacc) {
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {
      float v[16];
      tmem_load16(tmem + c * 16, v);
      if (c == 7) release();
      const int col = x.n + half * 128 + c * 16;
      stage_sums(staging, lane, x, v);
      if (lane == 0) {
        if (col < p.hidden && row < p.words) tma_store3(&p.out, staging, col, row, 0, p.row0 != 0);
        store_commit();
      }
    }
    return;
  }
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float v[32];
    tmem_load32(tmem + c * 32, v);
    if (c == 3) release();
    const int col = x.n + half * 128 + c * 32;
    // no row that counts: nothing was summed
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = x.steps != 0 ? __fmul_rn(v[i], scale) : 0.f;
    stage_bf16(staging, lane, v);
    if (lane == 0) {
      if (col < p.hidden && row < p.words) tma_store(&p.out, staging, col, (int)p.word0 + row);
      store_commit();
    }
  }
}

// At the end of a block that gave up a wait.  Its own tiles of the gradients were not all written, so it
// makes NaN of all that the launch writes of `dw` and, where its rows go straight out, of `dh`; other
// blocks may write theirs over that.
__device__ __forceinline__ void give_up(const GemmParams& p, int n_rows, bool dh, bool dw) {
  if (threadIdx.x == 0) {
    *reinterpret_cast<volatile int64_t*>(p.report + 1) = 1;
    *reinterpret_cast<volatile int*>(p.lost) = 1;
  }
  const int vecs = p.hidden >> 3;
  const uint4 nan = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
  if (dh)
    for (int k = 0; k < n_rows; ++k)
      for (int v = threadIdx.x; v < vecs; v += blockDim.x) reinterpret_cast<uint4*>(p.gh + (int64_t)p.index[k] * p.hidden)[v] = nan;
  if (dw) {
    uint4* to = reinterpret_cast<uint4*>(p.gw + p.word0 * p.hidden);
    for (int64_t v = threadIdx.x; v < (int64_t)p.words * vecs; v += blockDim.x) to[v] = nan;
  }
  __syncthreads();  // what follows is for whole warps
}

// --------------------------------------------------------------------- product
// LONG: the gradient of logits of several chains; an instance of its own, as the sums take registers
template <int PASS, bool LONG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
lce_product_kernel(const __grid_constant__ GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages], empty[kStages], done[2], drained[2];
  __shared__ uint32_t tmem_at;
  __shared__ int gave_up;
  __shared__ float2 row_part[2][4][PASS == kStats ? 128 : 1];  // by turn, columns and row
  __shared__ volatile int stop[8][2];  // of two epilogue warps of the same 32 rows, by turn
  const uint32_t stages = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t full0 = smem_addr(full), empty0 = smem_addr(empty), done0 = smem_addr(done), drained0 = smem_addr(drained);
  constexpr int kLength = PASS == kStats ? kChain : kGradChain;  // stages of a chain; kGrads has one a tile
  const bool chained = PASS == kStats ? p.hidden > kLength * kInner : LONG;

  if (threadIdx.x == 0) {
    gave_up = 0;
    for (int i = 0; i < 16; ++i) stop[i >> 1][i & 1] = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(done0 + 8 * i, 1);
      mbar_init(drained0 + 8 * i, chained ? 2 * kEpilogueWarps : kEpilogueWarps);  // of both CTAs
    }
    mbar_init_fence();
    prefetch_map(&p.a);
    prefetch_map(&p.b);
  }
  if (warp == 1) tmem_alloc_pair(smem_addr(&tmem_at), 512);
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tmem = tmem_at;

  grid_release();
  grid_wait();
  const int n_rows = *p.count;
  Plan plan{};
  plan.make<PASS>(p, n_rows, gridDim.x >> 1);
  const int pair = blockIdx.x >> 1;
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      const uint32_t lead_full0 = map_to_rank(full0, 0);
      int it = 0;
      for (int turn = 0, t; ok && (t = plan.pick<PASS>(pair, turn)) >= 0; ++turn) {
        const Tile x = plan.at<PASS>(p, t);
        const bool outer_a = PASS == kGrads && x.kind == 1, outer_b = PASS == kGrads;
        const CUtensorMap* ma = outer_a ? &p.a2 : &p.a;
        const CUtensorMap* mb = outer_a ? &p.b2 : &p.b;
        const int am = x.m + rank * 128, bn = x.n + rank * (x.narrow ? 64 : 128);
        // kLogitGrad: W's rows start at the piece; dh: so do the inner values of W
        const int b_row0 = PASS == kLogitGrad ? (int)p.word0 : 0, b_k0 = PASS == kGrads && x.kind == 0 ? (int)p.word0 : 0;
        for (int k = 0; k < x.steps; ++k, ++it) {
          const int s = it % kStages;
          if (!mbar_wait(empty0 + 8 * s, ((it / kStages) & 1) ^ 1, p.wait_limit)) { ok = false; break; }
          if (rank == 0) mbar_expect_tx(full0 + 8 * s, x.narrow ? 2 * kStageBytes - kHalfBytes : 2 * kStageBytes);
          const uint32_t at = stages + s * kStageBytes, bt = at + kHalfBytes, bar = lead_full0 + 8 * s;
          const int kk = x.k0 + k * kInner;
          if (outer_a) {
            tma_load_pair(at, ma, am, kk, bar);
            tma_load_pair(at + kHalfBytes / 2, ma, am + 64, kk, bar);
          } else {
            tma_load_pair(at, ma, kk, am, bar);
          }
          if (outer_b) {
            tma_load_pair(bt, mb, bn, b_k0 + kk, bar);
            if (!x.narrow) tma_load_pair(bt + kHalfBytes / 2, mb, bn + 64, b_k0 + kk, bar);
          } else {
            tma_load_pair(bt, mb, kk, b_row0 + bn, bar);
          }
        }
      }
      // every stage is released before this CTA may go: the last arrivals come from the partner
      for (int i = 0; i < kStages && ok; ++i, ++it) ok = mbar_wait(empty0 + 8 * (it % kStages), ((it / kStages) & 1) ^ 1, p.wait_limit);
      if (!ok) {  // copies that are still under way end within microseconds
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int it = 0, chains = 0;
      for (int mine = 0, t; ok && (t = plan.pick<PASS>(pair, mine)) >= 0; ++mine) {
        const Tile x = plan.at<PASS>(p, t);
        const bool outer_a = PASS == kGrads && x.kind == 1;
        constexpr bool outer_b = PASS == kGrads;
        const uint32_t idesc = instruction(kTile, x.narrow ? kTile / 2 : kTile, outer_a, outer_b);
        int k = 0;
        do {  // one chain; a tile of no stage has an empty one
          const int last = PASS != kGrads && k + kLength < x.steps ? k + kLength : x.steps;
          const uint32_t acc = chains & 1, d = tmem + acc * kTile;
          if (!mbar_wait(drained0 + 8 * acc, ((chains >> 1) & 1) ^ 1, p.wait_limit)) { ok = false; break; }
          fence_after();
          for (bool begun = false; k < last; ++k, ++it) {
            const int s = it % kStages;
            if (!mbar_wait(full0 + 8 * s, (it / kStages) & 1, p.wait_limit)) { ok = false; break; }
            fence_after();
            const uint32_t at = stages + s * kStageBytes, bt = at + kHalfBytes;
            const uint64_t da = outer_a ? operand(at, kHalfBytes / 2, 1024) : operand(at, 16, 1024);
            const uint64_t db = outer_b ? operand(bt, kHalfBytes / 2, 1024) : operand(bt, 16, 1024);
            // 16 inner values further: 32 bytes along a row, or 16 lines of 128 bytes
            const uint64_t step_a = outer_a ? 2048 >> 4 : 32 >> 4, step_b = outer_b ? 2048 >> 4 : 32 >> 4;
#pragma unroll
            for (int q = 0; q < kInner / 16; ++q) {
              mma_pair(d, da + q * step_a, db + q * step_b, idesc, begun);
              begun = true;
            }
            commit_pair(empty0 + 8 * s);
          }
          if (!ok) break;
          commit_pair(done0 + 8 * acc);
          ++chains;
        } while (ok && k < x.steps);
      }
    }
    __syncwarp();
  } else if ((PASS == kStats || LONG) && chained) {
    // warps 2 to 17: four rows of 32, four of 64 columns; the sums of a tile stay in registers
    const uint32_t staging = stages + kStages * kStageBytes + (warp - 2) * kStagingBytes;
    if (PASS == kLogitGrad) prepare_rows(p, n_rows, blockIdx.x * kEpilogueWarps + warp - 2, gridDim.x * kEpilogueWarps);
    const int quarter = warp & 3, part = (warp - 2) >> 2, in_cta = quarter * 32 + lane, mates = quarter + (part >> 1) * 4;
    const uint32_t lead_drained0 = map_to_rank(drained0, 0);
    int chains = 0;
    for (int mine = 0, t; (t = plan.pick<PASS>(pair, mine)) >= 0; ++mine) {
      const Tile x = plan.at<PASS>(p, t);
      const int row = x.m + (int)rank * 128 + in_cta, turn = mine & 1;
      const RowValues values = row_values<PASS>(p, row, n_rows);  // on their way while the products run
      float v[64];
      for (int k = 0; k < x.steps && ok; k += kLength, ++chains) {
        const uint32_t acc = chains & 1, at = tmem + acc * kTile + part * 64 + ((uint32_t)(quarter * 32) << 16);
        ok = mbar_wait(done0 + 8 * acc, (chains >> 1) & 1, p.wait_limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        if (k == 0) {
          tmem_load64(at, v);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float more[16];
            tmem_load16(at + c * 16, more);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[c * 16 + i] = __fadd_rn(v[c * 16 + i], more[i]);
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(lead_drained0 + 8 * acc);
      }
      if (PASS == kLogitGrad) {
        if (!ok) break;
        logit_grad_part(p, reinterpret_cast<float(&)[32]>(v[0]), x.n + part * 64, row, staging, lane, values, row < n_rows);
        logit_grad_part(p, reinterpret_cast<float(&)[32]>(v[32]), x.n + part * 64 + 32, row, staging, lane, values, row < n_rows);
        continue;
      }
      // The two warps of these rows and 128 columns join.  One that gave up comes here, too, and both
      // leave: what belongs to a turn is written again two turns later, when they have met once more.
      if (ok) row_part[turn][part][in_cta] = stats_of(v, x.n + part * 64, p.words, values.label);
      else stop[mates][turn] = 1;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + mates) : "memory");
      ok = stop[mates][turn] == 0;
      if (!ok) break;
      if ((part & 1) == 0 && row < n_rows)
        p.part[(int64_t)(x.n / 128 + (part >> 1)) * p.rows + row] = join2(row_part[turn][part][in_cta], row_part[turn][part + 1][in_cta]);
    }
    if (PASS != kStats && lane == 0) store_wait();
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = ((warp - 2) >> 2) & 1, group = (warp - 2) >> 3;
    const uint32_t lead_drained0 = map_to_rank(drained0, 0);
    const float scale = PASS == kGrads ? all_scale(p) : 1.f;
    const uint32_t staging = stages + kStages * kStageBytes + (warp - 2) * kStagingBytes;
    if (PASS == kLogitGrad) prepare_rows(p, n_rows, blockIdx.x * kEpilogueWarps + warp - 2, gridDim.x * kEpilogueWarps);
    for (int mine = group, t; (t = plan.pick<PASS>(pair, mine)) >= 0; mine += 2) {
      const Tile x = plan.at<PASS>(p, t);
      const uint32_t acc = group;
      const int row = x.m + (int)rank * 128 + quarter * 32 + lane;
      const RowValues values = row_values<PASS>(p, row, n_rows);  // on their way while the products run
      ok = mbar_wait(done0 + 8 * acc, (mine >> 1) & 1, p.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const uint32_t at = tmem + acc * kTile + half * 128 + ((uint32_t)(quarter * 32) << 16);
      const auto release = [&] {
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(lead_drained0 + 8 * acc);
      };
      if (PASS == kStats) {
        float2 both[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v[64];
          tmem_load64(at + c * 64, v);
          if (c == 1) release();
          both[c] = stats_of(v, x.n + half * 128 + c * 64, p.words, values.label);
        }
        if (row < n_rows) p.part[(int64_t)(x.n / 128 + half) * p.rows + row] = join2(both[0], both[1]);
      }
      if (PASS == kLogitGrad) logit_grad_tile(p, x, at, row, half, staging, lane, values, row < n_rows, release);
      if (PASS == kGrads && x.kind == 0) dh_tile(p, x, at, row, n_rows, half, scale, staging, lane, release);
      if (PASS == kGrads && x.kind == 1) dw_tile(p, x, at, row, half, scale, staging, lane, release);
    }
    if (PASS != kStats && lane == 0) store_wait();
    __syncwarp();
  }
  if (!ok) gave_up = 1;
  fence_before();
  __syncthreads();
  if (gave_up) give_up(p, n_rows, PASS == kGrads && p.want_dh && p.gh != nullptr, PASS == kGrads && p.want_dw && !p.wacc);
  cluster_sync();
  fence_after();
  if (warp == 1) tmem_free_pair(tmem, 512);
}

// ------------------------------------------------------------ joining the sums
struct JoinArgs {
  const float *picked, *inv;
  float *top, *rest, *miss;
  int* count;
  const int* lost;
  int reduction, parts;
  float* loss;  // null, of lce_few_kernel: a launch of its own joins
};
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float mn = fmaxf(m, m2), sh = finite_shift(mn);
  s = __fadd_rn(__fmul_rn(s, expf(__fsub_rn(m, sh))), __fmul_rn(s2, expf(__fsub_rn(m2, sh))));
  m = mn;
}
constexpr int kJoinLoads = 8;  // partials that a thread loads at a time
// A row's partials are always joined in the same order, so its loss does not depend on the rows beside it:
// slice i of kJoinSlices has every kJoinSlices-th partial from i on, and a warp joins the slices.
// A thread's K of the slices, 32 apart.
constexpr int kJoinSlices = 64;
template <int K>
__device__ __forceinline__ void join_slices(const float2* __restrict__ part, int64_t rows, int64_t row, int slice, int parts, float (&m)[K],
                                            float (&s)[K]) {
  for (int i = slice; i < parts; i += kJoinSlices * kJoinLoads) {
    float2 x[K][kJoinLoads];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int u = 0; u < kJoinLoads; ++u) {
        const int at = i + k * 32 + u * kJoinSlices;
        x[k][u] = at < parts ? __ldcg(part + (int64_t)at * rows + row) : make_float2(-INFINITY, 0.f);
      }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float mn = m[k];
#pragma unroll
      for (int u = 0; u < kJoinLoads; ++u) mn = fmaxf(mn, x[k][u].x);
      const float sh = finite_shift(mn);
      s[k] = __fmul_rn(s[k], expf(__fsub_rn(m[k], sh)));
#pragma unroll
      for (int u = 0; u < kJoinLoads; ++u) s[k] = __fadd_rn(s[k], __fmul_rn(x[k][u].y, expf(__fsub_rn(x[k][u].x, sh))));
      m[k] = mn;
    }
  }
}
// m, s: of slices `lane` and `lane + 32`; lane 0 gets the row's.
__device__ __forceinline__ void join_warp(float& m, float& s, float m2, float s2) {
  join(m, s, m2, s2);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m2 = __shfl_xor_sync(0xffffffffu, m, o);
    s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, m2, s2);
  }
}
// The loss of packed row `at` from the maximum and the sum of its other words; what backward needs.
__device__ __forceinline__ double finish_row(const JoinArgs& j, int64_t at, const int* index, const int* label, float m, float s) {
  const double z = j.picked[at], top = m, rest = s;
  const bool known = label[at] >= 0, lost = __ldcg(j.lost) != 0;  // loaded together
  double loss_of;
  // an infinite logit of the label's own has no loss, as in PyTorch
  if (!known | lost | (z == INFINITY)) loss_of = NAN;
  else if (z >= top) loss_of = log1p(rest * exp(top - z));
  else loss_of = top - z + log(rest + exp(z - top));
  j.top[at] = finite_shift(m);  // all others -inf: exp(-inf - 0) is 0
  j.rest[at] = m == -INFINITY ? 0.f : log2f(s);
  j.miss[at] = (float)-expm1(-loss_of);
  if (j.reduction == kLceNone) j.loss[index[at]] = (float)loss_of;
  return loss_of;
}

// ---------------------------------------------------------- product, few rows
// Up to kLceFewRows rows the products read W once and little else.  A pair's tile of 256 rows would
// spend most of its products on rows that are not there: one row of 128256 words took 166 us of
// them at 1.9 GHz and more where the clock is lower, against 163 us of reading.  Here the words
// (for dh: the hidden columns) are the 128 rows of a tile, one CTA's, and the packed rows its N
// columns: lanes of tensor memory are words, columns are rows.  A stage is 18 or 24 KB, 16 of
// them W, so that 12 or 9 stages keep more of W on its way.
// kLceFewRows is as far as the accumulators go.  The loss alone, and with gradients, us (in brackets as
// tiles of a pair): 128256 words of 4096, 17 rows 174, 718 (203, 812), 32 rows 195, 723 (235, 874), 64 rows
// 226, 768 (224, 898).  A small head is bound by the epilogue, which takes the rows one behind the
// other, and loses by it: 32000 words of 1024, 17 rows 32, 107 (34, 117), 32 rows 41, 117 (34, 118), 64
// rows 54 to 59, 126 to 135 (29 to 38, 104 to 129).
constexpr int kFewThreads = 64 + 128;
// The statistics' last block joins their sums itself, which saves a launch, where its four warps need
// two turns of 512 partials at most (32000 words of 1024, the loss alone, 8 rows: 28.6 us with the
// launch, so 23.5; 16 rows, four turns: 28.8 and 29.8).
constexpr bool few_join(int64_t rows, int64_t parts) { return (rows + 3) / 4 * ((parts + 511) / 512) <= 2; }
template <int N>
struct FewShape {
  static constexpr int kStage = kHalfBytes + N * 128, kCount = (220 * 1024) / kStage, kSmem = kCount * kStage + 1024;
  static constexpr int kAccs = 8, kColumns = kAccs * N;  // accumulators in tensor memory
};
// Stages of a chain of the statistics.  One row of 128256 words x 4096: 174 us without chains, 179 with
// four stages, 186 with two; the loss of a confident row up to 25, 1.0 and 0.8e-6 off 64 bits.
constexpr int kFewChain = 4;
// Of dh; the logits for backward have theirs of kGradChain.
constexpr int kFewSumChain = kLceSumTerms / kInner;
template <int N>
__device__ __forceinline__ void tmem_load_rows(uint32_t at, float (&v)[N]) {
  if constexpr (N == 16) {
    tmem_load16(at, v);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 32) tmem_load32(at + c, reinterpret_cast<float(&)[32]>(v[c]));
  }
}

template <int PASS, int N>
__global__ void __launch_bounds__(kFewThreads, 1)
lce_few_kernel(const __grid_constant__ GemmParams p, float* acc, const JoinArgs j) {
  using S = FewShape<N>;
  constexpr int kLength = PASS == kStats ? kFewChain : PASS == kLogitGrad ? kGradChain : kFewSumChain;  // stages of a chain
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[S::kCount], empty[S::kCount], done[S::kAccs], drained[S::kAccs];
  __shared__ uint32_t tmem_at;
  __shared__ int gave_up;
  __shared__ volatile int stop;  // of the epilogue warps
  __shared__ int label_of[N];
  __shared__ float top_of[N], rest_of[N], scale_of[N];
  __shared__ int row_of[N];
  __shared__ float2 warp_part[4][N];
  __shared__ double row_loss[PASS == kStats ? N : 1];
  const uint32_t stages = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = smem_addr(full), empty0 = smem_addr(empty), done0 = smem_addr(done), drained0 = smem_addr(drained);
  grid_release();
  grid_wait();
  const int n_rows = *p.count;
  if (threadIdx.x == 0) {
    gave_up = 0;
    stop = 0;
    for (int i = 0; i < S::kCount; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < S::kAccs; ++i) {
      mbar_init(done0 + 8 * i, 1);
      mbar_init(drained0 + 8 * i, 4);
    }
    mbar_init_fence();
    prefetch_map(&p.a);
    prefetch_map(&p.b);
  }
  if (PASS != kGrads && threadIdx.x < N) {
    const int r = threadIdx.x;
    label_of[r] = r < n_rows ? p.label[r] : -1;
    if (PASS == kLogitGrad) {
      top_of[r] = r < n_rows ? p.top[r] : 0.f;
      rest_of[r] = r < n_rows ? p.rest[r] : INFINITY;
    }
  }
  if (PASS == kGrads && p.gh != nullptr && threadIdx.x < n_rows) {
    const int r = threadIdx.x;
    row_of[r] = p.index[r];
    scale_of[r] = row_scale(p, r, all_scale(p));
  }
  if (warp == 1) tmem_alloc(smem_addr(&tmem_at), S::kColumns);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;

  // tiles of 128 words, or of 128 hidden columns and a share of the words
  const int across = ((PASS == kGrads ? p.hidden : p.words) + 127) / 128, total = PASS == kGrads ? across * p.splits : across;
  const int all_steps = ((PASS == kGrads ? p.words : p.hidden) + kInner - 1) / kInner;
  auto share = [&](int t, int& first) {  // the inner steps of tile t
    if (PASS != kGrads) {
      first = 0;
      return all_steps;
    }
    const int split = t / across;
    first = (int)((int64_t)all_steps * split / p.splits);
    return (int)((int64_t)all_steps * (split + 1) / p.splits) - first;
  };
  bool ok = true;
  if (warp == 0) {
    if (elect_one()) {
      int it = 0;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        int first;
        const int steps = share(t, first), m = t % across * 128;
        for (int k = 0; k < steps; ++k, ++it) {
          const int s = it % S::kCount, kk = (first + k) * kInner;
          if (!mbar_wait(empty0 + 8 * s, ((it / S::kCount) & 1) ^ 1, p.wait_limit)) { ok = false; break; }
          const uint32_t at = stages + s * S::kStage, bar = full0 + 8 * s;
          mbar_expect_tx(bar, S::kStage);
          if (PASS == kGrads) {
            tma_load(at, &p.a, m, (int)p.word0 + kk, bar);
            tma_load(at + kHalfBytes / 2, &p.a, m + 64, (int)p.word0 + kk, bar);
          } else {
            tma_load(at, &p.a, kk, (int)p.word0 + m, bar);
          }
          tma_load(at + kHalfBytes, &p.b, kk, 0, bar);
        }
      }
      if (!ok) {  // copies that are still under way end within microseconds
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = instruction(128, N, PASS == kGrads, false);
      int it = 0, chains = 0;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        int first;
        const int steps = share(t, first);
        int k = 0;
        do {  // one chain; a tile of no stage has an empty one
          const int last = k + kLength < steps ? k + kLength : steps;
          const uint32_t buf = chains % S::kAccs, d = tmem + buf * N;
          if (!mbar_wait(drained0 + 8 * buf, ((chains / S::kAccs) & 1) ^ 1, p.wait_limit)) { ok = false; break; }
          fence_after();
          for (bool begun = false; k < last; ++k, ++it) {
            const int s = it % S::kCount;
            if (!mbar_wait(full0 + 8 * s, (it / S::kCount) & 1, p.wait_limit)) { ok = false; break; }
            fence_after();
            const uint32_t at = stages + s * S::kStage;
            const uint64_t da = PASS == kGrads ? operand(at, kHalfBytes / 2, 1024) : operand(at, 16, 1024);
            const uint64_t db = operand(at + kHalfBytes, 16, 1024);
            constexpr uint64_t step_a = PASS == kGrads ? 2048 >> 4 : 32 >> 4;
#pragma unroll
            for (int q = 0; q < kInner / 16; ++q) {
              mma(d, da + q * step_a, db + q * (32 >> 4), idesc, begun);
              begun = true;
            }
            commit(empty0 + 8 * s);
          }
          if (!ok) break;
          commit(done0 + 8 * buf);
          ++chains;
        } while (ok && k < steps);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    int chains = 0;
    if (PASS == kLogitGrad) prepare_rows(p, n_rows, blockIdx.x * 4 + warp - 2, gridDim.x * 4);
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      int first;
      const int steps = share(t, first), m = t % across * 128;
      float v[N];
      int k = 0;
      do {
        const uint32_t buf = chains % S::kAccs, from = tmem + buf * N + ((uint32_t)(quarter * 32) << 16);
        ok = mbar_wait(done0 + 8 * buf, (chains / S::kAccs) & 1, p.wait_limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        if (k == 0) {
          tmem_load_rows<N>(from, v);
        } else {
          float more[N];
          tmem_load_rows<N>(from, more);
#pragma unroll
          for (int r = 0; r < N; ++r) v[r] = __fadd_rn(v[r], more[r]);
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(drained0 + 8 * buf);
        ++chains;
        k += kLength;
      } while (k < steps);
      if (PASS != kStats && !ok) break;
      const int at = m + quarter * 32 + lane;  // this lane's word of the piece, or hidden column
      if (PASS == kStats) {
        if (!ok) stop = 1;
        const bool in = at < p.words;
        float2 own = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int r = 0; r < N; ++r) {
          if (r >= n_rows) break;
          const float z = in && label_of[r] != at ? v[r] : -INFINITY;  // the label's is known apart
          float top = z;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          float sum = exp_of(__fsub_rn(z, finite_shift(top)));
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
          if (lane == (r & 31)) own = make_float2(top, sum);
          if ((r & 31) == 31 || r == n_rows - 1) {
            if (lane <= (r & 31)) warp_part[quarter][r - (r & 31) + lane] = own;
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the four epilogue warps; one that gave up, too, comes here
        ok = stop == 0;
        if (!ok) break;
        const int r = threadIdx.x - 64;
        if (r < n_rows) {
          p.part[(int64_t)(m / 128) * p.rows + r] = join2(join2(warp_part[0][r], warp_part[1][r]), join2(warp_part[2][r], warp_part[3][r]));
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");  // before warp_part is written again
      } else if (PASS == kLogitGrad) {
        const int word = (int)p.word0 + at;
        if (at < p.words) {
#pragma unroll
          for (int r = 0; r < N; ++r) {
            float d = label_of[r] == word ? -1.f : share_of(v[r], top_of[r], rest_of[r]);
            if (r >= n_rows) d = 0.f;  // the rows that pad the inner dimension of dW
            p.d[(int64_t)r * p.pitch + at] = (uint16_t)f32_to_bf16_rne_bits(d);
          }
          for (int r = N; r < kLceRowPad; ++r) p.d[(int64_t)r * p.pitch + at] = 0;
        }
      } else if (at < p.hidden && p.gh != nullptr) {  // one piece, one split: the whole sums
#pragma unroll
        for (int r = 0; r < N; ++r) {
          if (r >= n_rows) break;
          p.gh[(int64_t)row_of[r] * p.hidden + at] = (uint16_t)f32_to_bf16_rne_bits(__fmul_rn(v[r], scale_of[r]));
        }
      } else if (at < p.hidden) {
        float* to = acc + (int64_t)(t / across) * p.padded * p.row_pitch + at;
#pragma unroll
        for (int r = 0; r < N; ++r) {
          if (r >= n_rows) break;
          const float x = steps != 0 ? v[r] : 0.f;
          to[(int64_t)r * p.row_pitch] = p.first ? x : __fadd_rn(to[(int64_t)r * p.row_pitch], x);
        }
      }
    }
  }
  if (PASS == kStats && j.loss != nullptr && warp >= 2) {
    // The block that is the last to come here joins the sums of all of them.
    const int t = threadIdx.x - 64;
    if (!ok && t == 0) *reinterpret_cast<volatile int*>(p.lost) = 1;
    __threadfence();
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (t == 0) stop = atomicAdd(j.count + 1, 1) == (int)gridDim.x - 1;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (stop) {
      __threadfence();
      for (int r = t >> 5; r < n_rows; r += 4) {
        float m[2] = {-INFINITY, -INFINITY}, s[2] = {0.f, 0.f};
        join_slices(p.part, p.rows, r, lane, j.parts, m, s);
        join_warp(m[0], s[0], m[1], s[1]);
        if (lane == 0) warp_part[0][r] = make_float2(m[0], s[0]);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (t < n_rows) row_loss[t] = finish_row(j, t, p.index, p.label, warp_part[0][t].x, warp_part[0][t].y);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (t == 0 && j.reduction != kLceNone) {
        double sum = 0.0;
        for (int i = 0; i < n_rows; ++i) sum += row_loss[i];
        *j.loss = (float)(j.reduction == kLceMean ? sum * (double)*j.inv : sum);
      }
    }
  }
  if (!ok) gave_up = 1;
  fence_before();
  __syncthreads();
  if (gave_up) give_up(p, n_rows, PASS == kGrads && p.gh != nullptr, false);
  fence_after();
  if (warp == 1) tmem_free(tmem, S::kColumns);
}

// dW of few rows: W's size to write, and products of a single stage for each tile, 128 words by 256
// hidden columns.  What goes out in 256 bytes of a row at a time or more gets 6.1 TB/s, in the 128
// bytes of a tiled store 5.0, whatever computes it.  So four warps take a tile, each stages its 32 rows
// whole, 528 bytes apart (free of bank conflicts), and each lane copies one.  A CTA takes
// consecutive tiles along the rows of dW: d of its words stays in shared memory and is read once, the
// rows of h come out of L2 again and again.  32 rows, hidden 8192, 128256 words (h 1 MB, d 16 MB, dW
// 2.1 GB), on one GPU in turn: 1370 us for loss and gradients, about 375 of them here; with the rows of h
// kept and d read again, or in the pair kernel, 1460.
constexpr int kFewDwStages = 2, kFewDwRow = 528, kFewDwStaging = 32 * kFewDwRow, kFewDwWarps = 8, kFewDwThreads = 64 + 32 * kFewDwWarps;
constexpr int kFewDwSmem = kFewDwStages * 2 * kHalfBytes + kHalfBytes + kFewDwWarps * kFewDwStaging + 1024;
__global__ void __launch_bounds__(kFewDwThreads, 1)
lce_few_dw_kernel(const __grid_constant__ GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kFewDwStages], empty[kFewDwStages], done[2], drained[2], d_full[1], d_empty[1];
  __shared__ uint32_t tmem_at;
  __shared__ int gave_up;
  const uint32_t stages = (smem_addr(smem_raw) + 1023u) & ~1023u, d_at = stages + kFewDwStages * 2 * kHalfBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = smem_addr(full), empty0 = smem_addr(empty), done0 = smem_addr(done), drained0 = smem_addr(drained);
  const uint32_t d_full0 = smem_addr(d_full), d_empty0 = smem_addr(d_empty);
  if (threadIdx.x == 0) {
    gave_up = 0;
    for (int i = 0; i < kFewDwStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(done0 + 8 * i, 1);
      mbar_init(drained0 + 8 * i, kFewDwWarps / 2);
    }
    mbar_init(d_full0, 1);
    mbar_init(d_empty0, 1);
    mbar_init_fence();
    prefetch_map(&p.a2);
    prefetch_map(&p.b2);
  }
  if (warp == 1) tmem_alloc(smem_addr(&tmem_at), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;
  grid_release();
  grid_wait();

  const int across = (p.hidden + kTile - 1) / kTile, total = across * ((p.words + 127) / 128);
  const int begin = (int)((int64_t)total * blockIdx.x / gridDim.x), end = (int)((int64_t)total * (blockIdx.x + 1) / gridDim.x);
  const int first_m = begin / across;
  bool ok = true;
  if (warp == 0) {
    if (elect_one()) {
      int m = first_m, column = begin - first_m * across;
      for (int t = begin; t < end && ok; ++t) {
        if (t == begin || column == 0) {
          if (!mbar_wait(d_empty0, ((m - first_m) & 1) ^ 1, p.wait_limit)) { ok = false; break; }
          mbar_expect_tx(d_full0, kHalfBytes);
          tma_load(d_at, &p.a2, m * 128, 0, d_full0);
          tma_load(d_at + kHalfBytes / 2, &p.a2, m * 128 + 64, 0, d_full0);
        }
        const int n = t - begin, s = n % kFewDwStages;
        if (!mbar_wait(empty0 + 8 * s, ((n / kFewDwStages) & 1) ^ 1, p.wait_limit)) { ok = false; break; }
        mbar_expect_tx(full0 + 8 * s, 2 * kHalfBytes);
        for (int i = 0; i < 4; ++i)
          tma_load(stages + (s * 4 + i) * (kHalfBytes / 2), &p.b2, column * kTile + i * 64, 0, full0 + 8 * s);
        if (++column == across) column = 0, ++m;
      }
      if (!ok) {  // copies that are still under way end within microseconds
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = instruction(128, kTile, true, true);
      int m = first_m, column = begin - first_m * across;
      for (int t = begin; t < end && ok; ++t) {
        const int n = t - begin, s = n % kFewDwStages, acc = n & 1;
        if ((t == begin || column == 0) && !mbar_wait(d_full0, (m - first_m) & 1, p.wait_limit)) { ok = false; break; }
        if (!mbar_wait(drained0 + 8 * acc, ((n >> 1) & 1) ^ 1, p.wait_limit) || !mbar_wait(full0 + 8 * s, (n / kFewDwStages) & 1, p.wait_limit)) { ok = false; break; }
        fence_after();
        const uint64_t da = operand(d_at, kHalfBytes / 2, 1024), db = operand(stages + s * 2 * kHalfBytes, kHalfBytes / 2, 1024);
#pragma unroll
        for (int q = 0; q < kLceRowPad / 16; ++q) mma(tmem + acc * kTile, da + q * (2048 >> 4), db + q * (2048 >> 4), idesc, q > 0);
        commit(empty0 + 8 * s);
        commit(done0 + 8 * acc);
        if (++column == across) {
          commit(d_empty0);
          column = 0;
          ++m;
        }
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, group = (warp - 2) >> 2;
    const bool none = *p.count == 0;  // d and h are not there
    const float scale = all_scale(p);
    const uint32_t staging = d_at + kHalfBytes + (warp - 2) * kFewDwStaging;
    for (int t = begin + group; t < end; t += 2) {
      const int m = t / across, column = t - m * across;
      ok = mbar_wait(done0 + 8 * group, ((t - begin) >> 1) & 1, p.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const uint32_t at = tmem + group * kTile + ((uint32_t)(quarter * 32) << 16);
      store_wait_read();  // each lane its own row of the last tile
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        float v[32];
        tmem_load32(at + c * 32, v);
        if (c == 7) {
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(drained0 + 8 * group);
        }
        uint32_t out[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) out[i] = none ? 0u : f32x2_to_bf16x2_rne(__fmul_rn(v[2 * i], scale), __fmul_rn(v[2 * i + 1], scale));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st_shared16(staging + lane * kFewDwRow + c * 64 + i * 16, out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
      }
      store_fence();
      const int row = m * 128 + quarter * 32 + lane, col = column * kTile;
      if (row < p.words && col < p.hidden) {
        const int values = p.hidden - col < kTile ? p.hidden - col : kTile;
        bulk_store(p.gw + (p.word0 + row) * p.hidden + col, staging + lane * kFewDwRow, values * 2);
      }
      store_commit();
    }
    store_wait();
    __syncwarp();
  }
  if (!ok) gave_up = 1;
  fence_before();
  __syncthreads();
  if (gave_up) give_up(p, 0, false, true);
  fence_after();
  if (warp == 1) tmem_free(tmem, 512);
}

// ------------------------------------------------------------- packing of rows
constexpr int kScanThreads = 1024;

// index[k] = row of the k-th label that counts, label[k] = that label (-1: outside the vocabulary),
// count[0] = how many, count[1] = 0, inv, lost = 0; row_loss of ignored rows = 0.
__global__ void __launch_bounds__(kScanThreads)
lce_scan_kernel(const int64_t* __restrict__ labels, int64_t rows, int64_t vocab, int64_t ignore, int* index, int* label,
                int* count, float* inv, int* lost, float* row_loss, volatile int64_t* bad) {
  __shared__ int warps[kScanThreads / 32 + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int64_t r0 = 0; r0 < rows; r0 += kScanThreads) {
    const int64_t r = r0 + threadIdx.x;
    const int64_t lab = r < rows ? labels[r] : ignore;
    const bool in = lab != ignore;
    const unsigned mask = __ballot_sync(0xffffffffu, in);
    if (lane == 0) warps[warp] = __popc(mask);
    __syncthreads();
    if (warp == 0) {
      const int c = warps[lane];
      int x = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      warps[lane] = x - c;
      if (lane == 31) warps[32] = x;
    }
    __syncthreads();
    if (in) {
      const int k = base + warps[warp] + __popc(mask & ((1u << lane) - 1u));
      const bool known = lab >= 0 && lab < vocab;
      if (!known) bad[lab < 0 ? 2 : 0] = lab;
      index[k] = (int)r;
      label[k] = known ? (int)lab : -1;
    } else if (row_loss != nullptr && r < rows) {
      row_loss[r] = 0.f;
    }
    base += warps[32];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    count[0] = base;
    count[1] = *lost = 0;
    *inv = __fdiv_rn(1.f, (float)(base < 1 ? 1 : base));
  }
}

// packed[k] = h[index[k]], zero rows up to the next multiple of kLceRowPad, and the logit of its
// label.  THREADS a row: a warp, or a block where there are few rows (32 of 8192: 20 us with a warp).
constexpr int kPackThreads = 256, kPackRows = kPackThreads / 32;
struct PackArgs {
  const uint16_t* h;
  int64_t h_stride;
  const uint16_t* w;
  int64_t w_stride;
  int hidden;
  uint16_t* packed;
  int64_t packed_pitch;
  float* picked;
};
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {  // of two bf16 pairs
  c = __fmaf_rn(__uint_as_float(a << 16), __uint_as_float(b << 16), c);
  return __fmaf_rn(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u), c);
}
// n: how many rows are packed; `row`, `label`: of packed row k < n
template <int THREADS>
__device__ __forceinline__ void pack_row(const PackArgs& a, int64_t k, int n, int row, int label) {
  const int vecs = a.hidden >> 3, lane = threadIdx.x % THREADS;
  uint4* to = reinterpret_cast<uint4*>(a.packed + k * a.packed_pitch);
  if (k < n) {
    const uint4* from = reinterpret_cast<const uint4*>(a.h + row * a.h_stride);
    const uint4* word = reinterpret_cast<const uint4*>(a.w + (label < 0 ? 0 : label) * a.w_stride);
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int v = lane; v < vecs; v += THREADS) {
      const uint4 f = from[v], g = word[v];
      to[v] = f;
      x[0] = dot2(f.x, g.x, x[0]);
      x[1] = dot2(f.y, g.y, x[1]);
      x[2] = dot2(f.z, g.z, x[2]);
      x[3] = dot2(f.w, g.w, x[3]);
    }
    float z = __fadd_rn(__fadd_rn(x[0], x[1]), __fadd_rn(x[2], x[3]));
    if constexpr (THREADS == 32) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z = __fadd_rn(z, __shfl_xor_sync(0xffffffffu, z, o));
    } else {  // k is the whole block's
      __shared__ float red[THREADS / 32];
      z = block_sum<THREADS>(z, red);
    }
    if (lane == 0) a.picked[k] = z;
  } else if (k < (n + kLceRowPad - 1) / kLceRowPad * kLceRowPad) {
    for (int v = lane; v < vecs; v += THREADS) to[v] = make_uint4(0, 0, 0, 0);
  }
}
__global__ void __launch_bounds__(kPackThreads)
lce_pack_kernel(const PackArgs a, const int* __restrict__ index, const int* __restrict__ label, const int* __restrict__ count) {
  const int64_t k = (int64_t)blockIdx.x * kPackRows + (threadIdx.x >> 5);
  const int n = *count;
  pack_row<32>(a, k, n, k < n ? index[k] : 0, k < n ? label[k] : 0);
}

// Both in one launch for up to kScanPackRows rows: every block looks through all labels (32 KB at
// most, from L2) for the eight rows that it packs.  One row: 7 us, as two launches 13.
// Up to kScanPackBlockRows a row has a block, beyond a warp.  The loss of 256 words of 4096, us, with a
// block and with a warp: 32 rows 33 and 37, 512 rows 33.4 and 36.6, 768 rows 37.6 and 36.7, 1024 rows 40.0
// and 36.8.
constexpr int kScanPackRows = 4096, kScanPackBlockRows = 512;
template <int THREADS>
__global__ void __launch_bounds__(kPackThreads)
lce_scan_pack_kernel(const PackArgs a, const int64_t* __restrict__ labels, int rows, int64_t vocab, int64_t ignore, int* index,
                     int* label, int* count, float* inv, int* lost, float* row_loss, volatile int64_t* bad) {
  constexpr int kOwn = kPackThreads / THREADS, kEach = (THREADS == 32 ? kScanPackRows : kScanPackBlockRows) / kPackThreads;
  __shared__ int warps[kPackThreads / 32], source[kOwn], source_label[kOwn];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = blockIdx.x * kOwn;
  const int each = (rows + kPackThreads - 1) / kPackThreads, r0 = threadIdx.x * each;
  int64_t lab[kEach];
  int c = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    lab[i] = i < each && r0 + i < rows ? labels[r0 + i] : ignore;
    c += lab[i] != ignore;
  }
  int x = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warps[warp] = x;
  if (threadIdx.x < kOwn) source[threadIdx.x] = source_label[threadIdx.x] = 0;
  __syncthreads();
  int k = x - c, n = 0;
#pragma unroll
  for (int w = 0; w < kPackThreads / 32; ++w) {
    if (w < warp) k += warps[w];
    n += warps[w];
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int r = r0 + i;
    if (lab[i] != ignore) {
      if (k >= first && k < first + kOwn) {
        const bool known = lab[i] >= 0 && lab[i] < vocab;
        if (!known) bad[lab[i] < 0 ? 2 : 0] = lab[i];
        source[k - first] = index[k] = r;
        source_label[k - first] = label[k] = known ? (int)lab[i] : -1;
      }
      ++k;
    } else if (row_loss != nullptr && r >= first && r < first + kOwn && i < each && r < rows) {
      row_loss[r] = 0.f;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    count[0] = n;
    count[1] = *lost = 0;
    *inv = __fdiv_rn(1.f, (float)(n < 1 ? 1 : n));
  }
  __syncthreads();
  const int own = threadIdx.x / THREADS;
  pack_row<THREADS>(a, first + own, n, source[own], source_label[own]);
}

// A block has 8 rows (the partials of 4 are one 32-byte sector) and 64 slices of the words; a thread
// loads eight partials at a time.  One row of 128256 words: 1002 partials, 20 us with one load at a
// time in 32 slices.
constexpr int kJoinRows = 8, kJoinThreads = kJoinRows * kJoinSlices;
__global__ void __launch_bounds__(kJoinThreads)
lce_join_kernel(const float2* __restrict__ part, int64_t rows, const int* __restrict__ index, const int* __restrict__ label,
                const JoinArgs j, double* sums) {
  __shared__ float sm[kJoinSlices][kJoinRows], ss[kJoinSlices][kJoinRows];
  __shared__ double one[kJoinRows];
  __shared__ int is_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_release();
  grid_wait();
  const int n = *j.count, of = threadIdx.x % kJoinRows, slice = threadIdx.x / kJoinRows;
  const int64_t row = (int64_t)blockIdx.x * kJoinRows + of;
  float mine[1] = {-INFINITY}, sum[1] = {0.f};
  if (row < n) join_slices(part, rows, row, slice, j.parts, mine, sum);
  sm[slice][of] = mine[0];
  ss[slice][of] = sum[0];
  __syncthreads();
  if (warp < kJoinRows) {  // warp w finishes the block's row w
    float m = sm[lane][warp], s = ss[lane][warp];
    join_warp(m, s, sm[lane + 32][warp], ss[lane + 32][warp]);
    const int64_t at = (int64_t)blockIdx.x * kJoinRows + warp;
    if (lane == 0) {
      const double loss_of = at < n ? finish_row(j, at, index, label, m, s) : 0.0;
      one[warp] = loss_of;
    }
  }
  if (j.reduction == kLceNone) return;
  __syncthreads();
  if (threadIdx.x == 0) {  // the same order whatever the blocks' order
    double t = 0.0;
    for (int i = 0; i < kJoinRows; ++i) t += one[i];
    sums[blockIdx.x] = t;
    __threadfence();
    is_last = atomicAdd(j.count + 1, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (is_last && warp == 0) {
    __threadfence();
    double t = 0.0;
    for (int i = lane; i < (int)gridDim.x; i += 32) t += __ldcg(sums + i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) *j.loss = (float)(j.reduction == kLceMean ? t * (double)*j.inv : t);
  }
}

// -------------------------------------------------- dh: splits joined, rounded
// Rows whose label is ignored become zero.
__global__ void __launch_bounds__(128)
lce_join_grad_kernel(const float* __restrict__ acc, int splits, int64_t padded, int64_t pitch, const int* __restrict__ index,
                     const int64_t* __restrict__ labels, int64_t ignore, const int* __restrict__ count, int hidden,
                     const float* __restrict__ miss, const float* inv, const float* g, const int* lost, const float* row_g,
                     uint16_t* gh) {
  const int64_t k = blockIdx.x;
  const int col = (blockIdx.y * 128 + threadIdx.x) * 8;
  grid_wait();
  if (col >= hidden) return;
  if (labels[k] == ignore) *reinterpret_cast<uint4*>(gh + k * hidden + col) = make_uint4(0, 0, 0, 0);
  if (k >= *count) return;
  float scale = miss[k];
  if (*lost != 0) scale = NAN;
  if (inv != nullptr) scale = __fmul_rn(scale, *inv);
  if (g != nullptr) scale = __fmul_rn(scale, *g);
  if (row_g != nullptr) scale = __fmul_rn(scale, row_g[index[k]]);
  float v[8] = {};
  for (int s = 0; s < splits; ++s) {
    const V8 x = ld32(acc + ((int64_t)s * padded + k) * pitch + col);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], __uint_as_float(x.w[i]));
  }
  store_bf16x8(gh + (int64_t)index[k] * hidden + col, v, scale);
}

// ------------------------------------------------------- dW of many rows, rounded
// One piece, from its fp32 sums.
__global__ void __launch_bounds__(128)
lce_round_head_kernel(const float* __restrict__ acc, int64_t pitch, int hidden, const float* inv, const float* g, const int* lost,
                      uint16_t* gw) {
  const int64_t word = blockIdx.x;
  const int col = (blockIdx.y * 128 + threadIdx.x) * 8;
  grid_wait();
  if (col >= hidden) return;
  const float scale = all_scale(inv, g, lost);
  const V8 x = ld32(acc + word * pitch + col);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(x.w[i]);
  store_bf16x8(gw + word * hidden + col, v, scale);
}

// ------------------------------------------------------------------- launching
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// The encoder is a call of the driver and wants a context; a thread that has made no call of the
// runtime yet (one of autograd's) has none.
cudaError_t make_context_current() {
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  return e != cudaSuccess ? e : cudaSetDevice(device);
}

// The fp32 sums of dh as (hidden, rows, splits), of dW as (hidden, words, 1), in boxes of 16 columns and
// 32 lines.
bool encode_acc(CUtensorMap* map, float* base, int64_t hidden, int64_t pitch, int64_t lines, int splits) {
  const auto fn = encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)hidden, (cuuint64_t)lines, (cuuint64_t)splits};
  const cuuint64_t strides[2] = {(cuuint64_t)pitch * 4, (cuuint64_t)pitch * 4 * (cuuint64_t)lines};
  const cuuint32_t box[3] = {16, 32, 1}, steps[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Boxes of `width` (64 to read, 32 to write) contiguous values and `lines` lines of a bf16 matrix;
// what lies outside reads as zero and is not written.
bool encode(CUtensorMap* map, const void* base, int64_t inner, int64_t lines_all, int64_t stride, int lines, int width = 64) {
  const auto fn = encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)lines_all}, strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t box[2] = {(cuuint32_t)width, (cuuint32_t)lines}, steps[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, steps,
            CU_TENSOR_MAP_INTERLEAVE_NONE, width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Launches a kernel that touches no global memory before its grid_wait: its blocks come up while the last
// ones of the kernel before it in the stream still run, where that one lets them, as those of this file do.
// The first launch of a backward pass follows whatever ran last.
template <class... Args, class... Given>
cudaError_t launch_behind(void (*kernel)(Args...), dim3 grid, int threads, int smem, cudaStream_t st, const Given&... given) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &attr;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, Args(given)...);
}

// Once for each kernel and device.
cudaError_t allow_smem(std::atomic<uint64_t>& done, const void* kernel, int bytes) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t(1) << (device & 63);
  if ((done.load(std::memory_order_relaxed) & bit) != 0 && device < 64) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <int PASS, bool LONG = false>
cudaError_t launch_product(const GemmParams& p, int64_t tiles, cudaStream_t st) {
  if (tiles <= 0) return cudaSuccess;
  if (tiles > (int64_t(1) << 30)) return cudaErrorInvalidValue;
  constexpr int smem = smem_of(PASS != kStats);
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, (const void*)lce_product_kernel<PASS, LONG>, smem);
  if (e != cudaSuccess) return e;
  const int pairs = (int)(tiles < kNumSMs / 2 ? tiles : kNumSMs / 2);
  count_launch();
  return launch_behind(lce_product_kernel<PASS, LONG>, dim3(2 * pairs), kGemmThreads, smem, st, p);
}

template <int PASS, int N>
cudaError_t launch_few_of(const GemmParams& p, float* acc, const JoinArgs& j, int64_t tiles, cudaStream_t st) {
  constexpr int smem = FewShape<N>::kSmem;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, (const void*)lce_few_kernel<PASS, N>, smem);
  if (e != cudaSuccess) return e;
  count_launch();
  return launch_behind(lce_few_kernel<PASS, N>, dim3((unsigned)(tiles < kNumSMs ? tiles : kNumSMs)), kFewThreads, smem, st, p, acc, j);
}
// 16 columns keep three more stages in flight and shorten the epilogue; up to 64 rows otherwise.
constexpr int few_columns(int64_t rows) { return rows <= 16 ? 16 : kLceFewRows; }
template <int PASS>
cudaError_t launch_few(const GemmParams& p, float* acc, const JoinArgs& j, int64_t tiles, cudaStream_t st) {
  if (tiles > (int64_t(1) << 30)) return cudaErrorInvalidValue;
  return few_columns(p.rows) == 16 ? launch_few_of<PASS, 16>(p, acc, j, tiles, st) : launch_few_of<PASS, kLceFewRows>(p, acc, j, tiles, st);
}

cudaError_t launch_few_dw(const GemmParams& p, int64_t tiles, cudaStream_t st) {
  if (tiles > (int64_t(1) << 30)) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, (const void*)lce_few_dw_kernel, kFewDwSmem);
  if (e != cudaSuccess) return e;
  count_launch();
  return launch_behind(lce_few_dw_kernel, dim3((unsigned)(tiles < kNumSMs ? tiles : kNumSMs)), kFewDwThreads, kFewDwSmem, st, p);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

bool args_ok(const LceArgs& a) {
  // the sizes bound how long a tile takes, far below the limit of the waits
  return a.rows > 0 && a.rows <= kLceMaxRows && a.hidden > 0 && a.hidden <= kLceMaxHidden && a.hidden % 8 == 0 && a.vocab > 0 &&
         a.vocab <= kLceMaxVocab && a.w_stride % 8 == 0 && aligned16(a.w) && aligned16(a.packed) && a.report != nullptr &&
         a.w_stride < (int64_t(1) << 36);
}

// Nanoseconds.  The longest tile that the sizes allow takes milliseconds.
std::atomic<uint64_t> wait_limit{2000000000ull};

void common_params(GemmParams& p, const LceArgs& a) {
  p.count = a.count;
  p.rows = a.rows;
  p.padded = lce_padded(a.rows);
  p.hidden = (int)a.hidden;
  p.row_pitch = lce_row_pitch(a.hidden);
  p.report = a.report;
  p.lost = a.lost;
  p.wait_limit = wait_limit.load(std::memory_order_relaxed);
  p.label = a.label;
}

}  // namespace

uint64_t lce_wait_limit(uint64_t nanoseconds) { return wait_limit.exchange(nanoseconds); }

int64_t lce_part_floats(int64_t rows, int64_t vocab) {
  return 2 * rows * (rows <= kLceFewRows ? (vocab + 127) / 128 : 2 * tiles_of(vocab));
}
int64_t lce_sum_doubles(int64_t rows) { return (rows + kJoinRows - 1) / kJoinRows; }

cudaError_t launch_lce_forward(const LceArgs& a, int reduction, float* part, float* picked, double* sums, float* loss,
                               cudaStream_t st) {
  if (!args_ok(a) || a.h_stride % 8 != 0 || !aligned16(a.h)) return cudaErrorInvalidValue;
  float* const row_loss = reduction == kLceNone ? loss : nullptr;
  const unsigned blocks = (unsigned)(lce_padded(a.rows) / kPackRows);
  const PackArgs k{(const uint16_t*)a.h, a.h_stride, (const uint16_t*)a.w, a.w_stride, (int)a.hidden, (uint16_t*)a.packed, lce_row_pitch(a.hidden), picked};
  if (a.rows <= kScanPackBlockRows) {
    count_launch();
    lce_scan_pack_kernel<kPackThreads><<<(unsigned)lce_padded(a.rows), kPackThreads, 0, st>>>(
        k, a.labels, (int)a.rows, a.vocab, a.ignore, a.index, a.label, a.count, a.inv, a.lost, row_loss, a.report);
  } else if (a.rows <= kScanPackRows) {
    count_launch();
    lce_scan_pack_kernel<32><<<blocks, kPackThreads, 0, st>>>(k, a.labels, (int)a.rows, a.vocab, a.ignore, a.index, a.label, a.count,
                                                              a.inv, a.lost, row_loss, a.report);
  } else {
    count_launch(2);
    lce_scan_kernel<<<1, kScanThreads, 0, st>>>(a.labels, a.rows, a.vocab, a.ignore, a.index, a.label, a.count, a.inv, a.lost, row_loss,
                                                a.report);
    lce_pack_kernel<<<blocks, kPackThreads, 0, st>>>(k, a.index, a.label, a.count);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || (e = make_context_current()) != cudaSuccess) return e;
  GemmParams p{};
  common_params(p, a);
  p.words = (int)a.vocab;
  p.part = reinterpret_cast<float2*>(part);
  const bool few = a.rows <= kLceFewRows;
  p.index = a.index;
  JoinArgs j{picked, a.inv, a.top, a.rest, a.miss, a.count, a.lost, reduction, (int)(few ? (a.vocab + 127) / 128 : 2 * tiles_of(a.vocab)), loss};
  if (few) {
    if (!encode(&p.a, a.w, a.hidden, a.vocab, a.w_stride, 128) ||
        !encode(&p.b, a.packed, a.hidden, p.padded, p.row_pitch, few_columns(a.rows)))
      return cudaErrorInvalidValue;
    const bool own = few_join(a.rows, j.parts);
    JoinArgs none{};
    e = launch_few<kStats>(p, nullptr, own ? j : none, j.parts, st);
    if (e != cudaSuccess || own) return e;
  } else {
    if (!encode(&p.a, a.packed, a.hidden, p.padded, p.row_pitch, 128) || !encode(&p.b, a.w, a.hidden, a.vocab, a.w_stride, 128))
      return cudaErrorInvalidValue;
    e = launch_product<kStats>(p, tiles_of(a.rows) * tiles_of(a.vocab), st);
  }
  if (e != cudaSuccess) return e;
  count_launch();
  return launch_behind(lce_join_kernel, dim3((unsigned)lce_sum_doubles(a.rows)), kJoinThreads, 0, st, p.part, a.rows, a.index, a.label, j,
                       sums);
}

int64_t lce_default_piece(int64_t rows, int64_t vocab) {
  const int64_t words = (int64_t(256) << 20) / (2 * lce_padded(rows)) / kTile * kTile;
  const int64_t all = tiles_of(vocab) * kTile;
  const int64_t most = words < all ? words : all;
  return most < kTile ? kTile : most < kLceMaxPiece ? most : kLceMaxPiece;
}

int lce_splits(int64_t rows, int64_t hidden, int64_t vocab, int64_t piece) {
  const int64_t words = piece < vocab ? piece : vocab, steps = words / kInner;
  if (vocab <= piece && steps <= 32) return 1;  // up to 9 us; a launch to join the splits is longer
  if (rows <= kLceFewRows) {
    // the number that leaves the fewest SMs idle in the last round; each split is as much again
    // of rows x hidden to write and read
    const int64_t across = (hidden + 127) / 128;
    int best = 1;
    double most = 0.0;
    for (int s = 1; s <= 16 && (s == 1 || s <= steps / 8); ++s) {
      const int64_t tiles = across * s, rounds = (tiles + kNumSMs - 1) / kNumSMs;
      const double busy = (double)tiles / (double)(rounds * kNumSMs);
      if (busy > most + 0.02) most = busy, best = s;
    }
    return best;
  }
  const int64_t tiles = tiles_of(rows) * tiles_of(hidden);
  int64_t s = kNumSMs / 2 / tiles;
  if (s > steps / 8) s = steps / 8;
  const int64_t least = (words + kLceSumTerms - 1) / kLceSumTerms;  // 16 at most
  return (int)(s < least ? least : s);
}

cudaError_t launch_lce_backward(const LceArgs& a, const LceGrad& g, cudaStream_t st) {
  if (!args_ok(a) || g.piece <= 0 || g.piece % kTile != 0 || g.piece > kLceMaxPiece || g.splits < 1 || g.g == nullptr) return cudaErrorInvalidValue;
  if (g.gh == nullptr && g.gw == nullptr) return cudaSuccess;
  if (g.d == nullptr || (g.gh != nullptr && g.acc == nullptr && !lce_direct(a.vocab, g.piece, g.splits)) || (g.gw != nullptr && g.scaled == nullptr) ||
      (g.gw != nullptr && g.wacc == nullptr && lce_row_groups(a.rows) > 1)) return cudaErrorInvalidValue;
  cudaError_t e = make_context_current();
  if (e != cudaSuccess) return e;
  const int64_t pieces = lce_pieces(a.vocab, g.piece), pitch = lce_piece_pitch(a.vocab, g.piece);
  GemmParams p{};
  common_params(p, a);
  p.top = a.top;
  p.rest = a.rest;
  p.miss = a.miss;
  p.row_g = g.reduction == kLceNone ? g.g : nullptr;
  p.index = a.index;
  p.packed = (const uint16_t*)a.packed;
  p.scaled = g.gw != nullptr ? (uint16_t*)g.scaled : nullptr;
  GemmParams q{};
  common_params(q, a);
  q.inv = g.reduction == kLceMean ? a.inv : nullptr;
  q.g = g.reduction == kLceNone ? nullptr : g.g;
  const bool direct = lce_direct(a.vocab, g.piece, g.splits);
  p.gh = q.gh = direct ? (uint16_t*)g.gh : nullptr;
  p.labels = a.labels;
  p.ignore = a.ignore;
  q.miss = a.miss;
  q.index = a.index;
  q.row_g = p.row_g;
  q.want_dh = g.gh != nullptr;
  q.want_dw = g.gw != nullptr;
  q.gw = (uint16_t*)g.gw;
  const int groups = q.want_dw ? (int)lce_row_groups(a.rows) : 1;
  q.wacc = groups > 1;
  q.splits = g.splits;
  // few rows: `few` has the operands of dh, q those of dW alone
  const bool is_few = a.rows <= kLceFewRows;
  const int columns = few_columns(a.rows);
  GemmParams few = q;
  if (is_few) q.want_dh = 0;
  p.d = (uint16_t*)g.d;
  p.pitch = pitch;
  if (!encode(is_few ? &p.b : &p.a, a.packed, a.hidden, p.padded, p.row_pitch, is_few ? columns : 128) ||
      !encode(is_few ? &p.a : &p.b, a.w, a.hidden, a.vocab, a.w_stride, 128) ||
      !encode(is_few ? &few.a : &q.b, a.w, a.hidden, a.vocab, a.w_stride, 64) || (q.want_dw && !encode(&q.b2, g.scaled, a.hidden, p.padded, p.row_pitch, 64)) ||
      (q.want_dw && !is_few && !q.wacc && !encode(&q.out, g.gw, a.hidden, a.vocab, a.hidden, 32, 32)) ||
      (q.want_dh && !direct && !encode_acc(&q.out_acc, g.acc, a.hidden, p.row_pitch, p.padded, g.splits)))
    return cudaErrorInvalidValue;
  for (int64_t i = 0; i < pieces; ++i) {
    p.word0 = q.word0 = i * g.piece;
    p.words = q.words = (int)(a.vocab - p.word0 < g.piece ? a.vocab - p.word0 : g.piece);
    q.first = i == 0;
    if (!encode(&q.a2, g.d, q.words, p.padded, pitch, 64)) return cudaErrorInvalidValue;
    if (is_few) {
      few.word0 = q.word0;
      few.words = q.words;
      few.first = q.first;
      if (!encode(&few.b, g.d, q.words, p.padded, pitch, columns)) return cudaErrorInvalidValue;
      if ((e = launch_few<kLogitGrad>(p, nullptr, JoinArgs{}, (p.words + 127) / 128, st)) != cudaSuccess) return e;
      if (few.want_dh && (e = launch_few<kGrads>(few, g.acc, JoinArgs{}, (a.hidden + 127) / 128 * g.splits, st)) != cudaSuccess) return e;
    } else {
      if (!encode(&p.out, g.d, q.words, p.padded, pitch, 32, 32) || !encode(&q.a, g.d, q.words, p.padded, pitch, 128))
        return cudaErrorInvalidValue;
      const int64_t tiles = tiles_of(a.rows) * tiles_of(p.words);
      e = a.hidden > kGradChain * kInner ? launch_product<kLogitGrad, true>(p, tiles, st) : launch_product<kLogitGrad>(p, tiles, st);
      if (e != cudaSuccess) return e;
    }
    p.scaled = p.gh = nullptr;  // the first piece has done it
    if (is_few) {
      if (q.want_dw && (e = launch_few_dw(q, (q.words + 127) / 128 * tiles_of(a.hidden), st)) != cudaSuccess) return e;
      continue;
    }
    const int64_t dh = g.gh != nullptr ? tiles_of(a.rows) * tiles_of(a.hidden) * g.splits : 0;
    const int64_t dw = q.want_dw ? tiles_of(q.words) * tiles_of(a.hidden) : 0;
    if (q.wacc && !encode_acc(&q.out, g.wacc, a.hidden, p.row_pitch, q.words, 1)) return cudaErrorInvalidValue;
    for (int k = 0; k < groups; ++k) {  // the first one takes dh, too
      q.row0 = k * kLceSumTerms;
      q.want_dh = k == 0 && g.gh != nullptr;
      if ((e = launch_product<kGrads>(q, (k == 0 ? dh : 0) + dw, st)) != cudaSuccess) return e;
    }
    if (q.wacc) {
      count_launch();
      e = launch_behind(lce_round_head_kernel, dim3((unsigned)q.words, (unsigned)((a.hidden + 1023) / 1024)), 128, 0, st, g.wacc, p.row_pitch,
                        (int)a.hidden, q.inv, q.g, a.lost, (uint16_t*)g.gw + q.word0 * a.hidden);
      if (e != cudaSuccess) return e;
    }
  }
  if (g.gh != nullptr && !direct) {
    count_launch();
    e = launch_behind(lce_join_grad_kernel, dim3((unsigned)a.rows, (unsigned)((a.hidden + 1023) / 1024)), 128, 0, st, g.acc, g.splits,
                      p.padded, p.row_pitch, a.index, a.labels, a.ignore, a.count, (int)a.hidden, a.miss, q.inv, q.g, a.lost, p.row_g,
                      (uint16_t*)g.gh);
  }
  return e;
}

}  // namespace oab
