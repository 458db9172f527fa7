// Host-side launch interface of the global gradient norm and clipping (clip_ops.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace oab {

enum ClipDtype : int { kClipBF16 = 0, kClipF16 = 1, kClipF32 = 2 };
enum ClipNorm : int { kNormL2 = 0, kNormL1 = 1, kNormInf = 2 };

// One gradient: n values one behind the other, at any element of its type.
struct ClipEntry {
  void* p;
  int64_t n;
  uint32_t dtype;
  uint32_t first_chunk;  // filled in by the launch
};
// Tensors of a launch; the table travels as a kernel argument, 32 KB at most, and costs the host
// its size: the tables are of 4, 11 and 31 KB.
constexpr int kClipFew = 160, kClipSome = 448, kClipMany = 1300;

// Doubles that the launches below need for `count` tensors: one partial per block.
int64_t clip_partials(int64_t count);
// The norm over all tensors.  out[0] = min(1, max_norm / (norm + 1e-6)), out[1] = norm.
// With `scale`, every value is then multiplied by out[0] in fp32 and rounded once, in place;
// nothing is touched where out[0] is 1.
cudaError_t launch_grad_norm(const ClipEntry* entries, int64_t count, int norm, float max_norm, bool scale, double* partials,
                             float* out, cudaStream_t st);
// The second half alone: coef is read from the device.
cudaError_t launch_grad_scale(const ClipEntry* entries, int64_t count, const float* coef, cudaStream_t st);

}  // namespace oab
