// The mixers' kernels of one element type (-DROSA_MIXER_TYPE, -DROSA_MIXER_NAME): one translation
// unit per type and operator (-DROSA_MIXER_WINDOW), so that they build side by side.
#if ROSA_MIXER_WINDOW
#include "window_attention.hpp"
#else
#include "decay_attention.hpp"
#endif

#define ROSA_JOIN_(a, b) a##_##b
#define ROSA_JOIN(a, b) ROSA_JOIN_(a, b)

namespace rosa_mixer {

#if ROSA_MIXER_WINDOW
void ROSA_JOIN(window_forward, ROSA_MIXER_NAME)(const WindowCall& call) {
  window_forward<ROSA_MIXER_TYPE>(call);
}
void ROSA_JOIN(window_backward, ROSA_MIXER_NAME)(const WindowCall& call) {
  window_backward<ROSA_MIXER_TYPE>(call);
}
void ROSA_JOIN(window_update, ROSA_MIXER_NAME)(const WindowCall& call) {
  window_update<ROSA_MIXER_TYPE>(call);
}
#else
void ROSA_JOIN(decay_forward, ROSA_MIXER_NAME)(const DecayCall& call) {
  decay_forward<ROSA_MIXER_TYPE>(call);
}
void ROSA_JOIN(decay_backward, ROSA_MIXER_NAME)(const DecayCall& call) {
  decay_backward<ROSA_MIXER_TYPE>(call);
}
void ROSA_JOIN(decay_update, ROSA_MIXER_NAME)(const DecayCall& call) {
  decay_update<ROSA_MIXER_TYPE>(call);
}
#endif

}  // namespace rosa_mixer
