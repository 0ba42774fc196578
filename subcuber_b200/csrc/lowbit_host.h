// Arguments of the products with an operand held in few bits (w4.cu, act8.cu).
#pragma once
#include "sw_host.h"

namespace sb200 {
namespace lowbit {

// Weights in format W4 (lowbit_format.cuh); zeros == nullptr: symmetric.
struct W4 {
  DType dtype;  // of the scales and of the activations: kF16 or kBF16
  int n, k, group;
  const void* codes;
  const void* scales;
  const void* zeros;
};

// Activations in format ACT8; rows of codes start every `pitch` bytes, rows of exponents every `exp_pitch`.
struct Act8 {
  DType dtype;  // of the activations and of dY: kF16 or kBF16
  int m, k;
  const void* codes;
  long long pitch;
  const void* exps;
  long long exp_pitch;
};

}  // namespace lowbit
}  // namespace sb200
