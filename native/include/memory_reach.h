// Host: whether an operator's outputs may share memory with its operands (gemm_group.hip, quant_block.hip).
#pragma once

#include <stdint.h>

namespace {

// What an entry answers, having launched nothing, where an output's memory reaches into an operand's: a workgroup could read
// what another has written. Tensors whose memory meshes without meeting are for the caller to tell apart.
constexpr int kMayShare = -2;

// A tensor's memory from its first byte to behind its last, which is that of element `last` (strides are not negative).
struct MemoryReach {
  unsigned __int128 first, end;

  MemoryReach(const void* p, bool empty, __int128 last, int size) : first((uintptr_t)p), end(empty ? first : first + (last + 1) * size) {}
  bool meets(const MemoryReach& o) const { return first < end && o.first < o.end && first < o.end && o.first < end; }
};

}  // namespace
