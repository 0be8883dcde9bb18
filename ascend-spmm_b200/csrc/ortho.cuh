// Shared by the two forms of the orthogonalised update (ortho.cu, ortho_small.cu).
#pragma once

namespace spmmb {

// Stored fp16 operand = value * scale.  Singular values are of order one, so
// a matrix's elements are of order 1 / sqrt(size): the scales keep them out
// of fp16's subnormals and leave a factor of 100 below its maximum.
constexpr float kScaleX = 512.f, kScaleG = 256.f, kScaleP = 256.f;

}  // namespace spmmb
