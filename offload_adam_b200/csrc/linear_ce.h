// Host-side launch interface of the cross-entropy kernels that keep no logits (linear_ce.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace oab {

constexpr int kLceTile = 256;     // rows and columns of an output tile; a piece of the vocabulary is a multiple
constexpr int kLceFewRows = 64;   // up to here the rows are the narrow side of the products
constexpr int kLceRowPad = 64;    // the packed rows are padded with zeros to a multiple of this
constexpr int kLceSumTerms = 65536;  // that an accumulator of the tensor cores sums
// Sizes that the kernels take.
constexpr int64_t kLceMaxRows = int64_t(1) << 24, kLceMaxHidden = int64_t(1) << 18, kLceMaxVocab = int64_t(1) << 26;
constexpr int64_t kLceMaxPiece = int64_t(1) << 20;  // words at a time

// Operands and workspaces of one loss.  `rows` are the rows of h; the kernels work on those whose
// label counts, packed in order: how many there are is known on the device only.
struct LceArgs {
  const void* h = nullptr;           // bf16 (rows, hidden), unit column stride; forward only
  int64_t h_stride = 0;              // elements, a multiple of 8; h is 16-byte aligned
  const void* w = nullptr;           // bf16 (vocab, hidden), likewise
  int64_t w_stride = 0;
  const int64_t* labels = nullptr;   // (rows,) contiguous
  int64_t rows = 0, hidden = 0, vocab = 0, ignore = -100;
  // kept from forward to backward
  int* index = nullptr;              // (rows,) packed row -> row
  int* label = nullptr;              // (rows,) label of the packed row, -1: outside the vocabulary
  int* count = nullptr;              // [0] packed rows, [1] ticket
  float* inv = nullptr;              // 1 / max(1, packed rows)
  int* lost = nullptr;               // not 0: a kernel gave up a wait, the loss and gradients are NaN
  float* top = nullptr;              // (rows,) largest logit of the packed row without its label, 0 where that is -inf
  float* rest = nullptr;             // (rows,) log2 of the sum of exp(logit - top) over the same words
  float* miss = nullptr;             // (rows,) 1 - probability of its label
  void* packed = nullptr;            // bf16 (rows padded, lce_row_pitch)
  int64_t* report = nullptr;         // host memory: [0] a label past the vocabulary, [1] a wait that gave up, [2] a negative label
};

// Rows of `packed` and of a piece of the logits' gradient.
inline int64_t lce_padded(int64_t rows) { return (rows + kLceRowPad - 1) / kLceRowPad * kLceRowPad; }

// Values from one of their rows to the next: whole 128-byte lines, which TMA reads and writes faster
// (640 rows of 840: the statistics 45 us, of 832 or 896 37), whatever the pitch of h is.
inline int64_t lce_row_pitch(int64_t hidden) { return (hidden + 63) / 64 * 64; }

enum LceReduction : int { kLceNone = 0, kLceMean = 1, kLceSum = 2 };

// How long a wait of the kernels for their own pipeline may take from now on; what it was.  0: none waits,
// every launch gives up.
uint64_t lce_wait_limit(uint64_t nanoseconds);

// Floats of `part` and doubles of `sums` that the forward pass needs.
int64_t lce_part_floats(int64_t rows, int64_t vocab);
int64_t lce_sum_doubles(int64_t rows);
// loss: one float, or one per row (kLceNone).  picked: (rows,) floats.
cudaError_t launch_lce_forward(const LceArgs& a, int reduction, float* part, float* picked, double* sums, float* loss,
                               cudaStream_t st);

struct LceGrad {
  int reduction = kLceMean;
  const float* g = nullptr;   // incoming gradient: one float, or one per row (kLceNone)
  void* gh = nullptr;         // bf16 (rows, hidden) contiguous, or null
  void* gw = nullptr;         // bf16 (vocab, hidden) contiguous, or null
  int64_t piece = 0;          // words at a time, a multiple of kLceTile
  void* d = nullptr;          // bf16 (padded rows, lce_piece_pitch)
  void* scaled = nullptr;     // bf16 (padded rows, lce_row_pitch), for gw
  int splits = 1;             // of the sum over the words in gh
  float* acc = nullptr;       // fp32 (splits, padded rows, lce_row_pitch), for gh unless lce_direct
  float* wacc = nullptr;      // fp32 (words of a piece, lce_row_pitch), for gw of several row groups
};
// Launches whose sums make up one gw.
inline int64_t lce_row_groups(int64_t rows) { return (rows + kLceSumTerms - 1) / kLceSumTerms; }
inline int64_t lce_pieces(int64_t vocab, int64_t piece) { return (vocab + piece - 1) / piece; }
inline int64_t lce_piece_pitch(int64_t vocab, int64_t piece) { return ((vocab < piece ? vocab : piece) + 63) / 64 * 64; }
// gh goes straight out: its sums are whole after one launch.
inline bool lce_direct(int64_t vocab, int64_t piece, int splits) { return vocab <= piece && splits == 1; }
// Words at a time, and splits, when the caller leaves them to the package.
int64_t lce_default_piece(int64_t rows, int64_t vocab);
int lce_splits(int64_t rows, int64_t hidden, int64_t vocab, int64_t piece);
cudaError_t launch_lce_backward(const LceArgs& a, const LceGrad& g, cudaStream_t st);

}  // namespace oab
