#include "categorical_sample_device.hpp"

template void mdp::launch_sample<mdp::bf16, false>(const mdp::SampleArgs&, hipStream_t);
template void mdp::launch_sample<mdp::bf16, true>(const mdp::SampleArgs&, hipStream_t);
