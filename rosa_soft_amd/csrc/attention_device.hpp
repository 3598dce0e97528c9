// What the softmax attention kernels share: the window's over inputs and ring caches, and the paged
// cache's.
#pragma once

#include "mixer_device.hpp"

namespace rosa_mixer {

constexpr int kKeys = 64;  // keys of a tile

// Waves per SIMD that a kernel is compiled for: two, so that products of one overlap the softmax
// of the other and accumulators share the registers that the rest can use directly; float32 tiles
// of 128 columns leave room in LDS for one block, and moving 128 columns element by element takes
// more registers.
template <typename T, int WIDTH, bool WHOLE>
constexpr int kWaves = WIDTH == 128 && (sizeof(T) == 4 || !WHOLE) ? 1 : 2;
constexpr float kLog2e = 1.4426950408889634f;

// Tiles in LDS of the training kernels.  Two of 16 bits, in turn: a wave stores the next while
// others work on the one before, and one barrier for a tile is enough (it lets no wave past that
// has not finished the tile before last).  One of float32, whose three planes leave no room.
template <typename T> constexpr int kBuffers = sizeof(T) == 2 ? 2 : 1;

// Weights are formed as 2^kLift p and rounded so: float16 would lose bits of a weight below 2^-14,
// which a long window's are.
template <typename T> constexpr float kLift = kNarrow<T> ? 8.0f : 0.0f;
template <typename T> constexpr float kUnlift = kNarrow<T> ? 1.0f / 256.0f : 1.0f;

// How far, in exponents of two, a score may pass the reference of its softmax before the sums so
// far are scaled to a new one: weights up to 2^kSlack (with kLift below float16's largest) are as
// exact, and most tiles leave the sums alone.
constexpr float kSlack = 6.0f;

// Whether two tiles of 16 tokens of a wave fit its registers.
template <typename T, int WIDTH> constexpr bool kPairs = !(sizeof(T) == 4 && WIDTH == 128);

}  // namespace rosa_mixer
