// camal_act_wgrad4.hip — the weight-gradient kernels whose workgroups take 4 co tiles of 32.
#include "camal_act_wgrad.hpp"

namespace camal {
template int act_wgrad_launch<4>(hipStream_t, const ActPlan&, const float*, const ActIn&, float*, ActOut, float*, int, int, int);
}
