#include "categorical_sample_device.hpp"

template void mdp::launch_sample<float, false>(const mdp::SampleArgs&, hipStream_t);
template void mdp::launch_sample<float, true>(const mdp::SampleArgs&, hipStream_t);
