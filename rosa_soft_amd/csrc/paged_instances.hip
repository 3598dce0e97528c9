// The kernels of the paged cache of one element type (-DROSA_MIXER_TYPE, -DROSA_MIXER_NAME): one
// translation unit per type, so that they build side by side.
#include "paged_attention.hpp"

#define ROSA_JOIN_(a, b) a##_##b
#define ROSA_JOIN(a, b) ROSA_JOIN_(a, b)

namespace rosa_mixer {

void ROSA_JOIN(paged_update, ROSA_MIXER_NAME)(const PagedCall& call) {
  paged_update<ROSA_MIXER_TYPE>(call);
}

}  // namespace rosa_mixer
