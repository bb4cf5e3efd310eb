// The prompt-attention kernel for head dimensions 64 and 128 (dense_narrow.cu).
#pragma once
#include "dense_common.cuh"

namespace dense {

constexpr int NARROW_BN = 64;              // keys per tile: the box of the K and V maps

// mq: box {64, group, 128 / group}; mk, mv: box {64, 1, NARROW_BN}.
int launch_narrow(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const Args& a, int head_dim,
                  bool f16, int mode, cudaStream_t st);

}  // namespace dense
