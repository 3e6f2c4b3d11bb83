// Which of a ring's copies may be in flight: turn u of a CTA uses stage
// u % stages, whose barrier then completes its phase of parity (u / stages) & 1.
// The copies of turns 0 .. stages - 1 are asked for ahead of the first turn, those
// of turn u + stages once turn u's have been met and read.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

namespace kda {

struct RingTurns {
    int32_t stages;

    __host__ __device__ int32_t stage(int32_t turn) const { return turn % stages; }
    __host__ __device__ uint32_t parity(int32_t turn) const { return static_cast<uint32_t>(turn / stages) & 1u; }
    // The turns whose copies may be in flight where turn `turn`'s were not met: [turn, end).
    __host__ __device__ int32_t end_in_flight(int32_t turn) const { return turn + stages; }
};

}  // namespace kda
