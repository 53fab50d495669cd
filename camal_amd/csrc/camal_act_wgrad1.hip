// camal_act_wgrad1.hip — the weight-gradient kernels whose workgroups take 1 co tile of 32.
#include "camal_act_wgrad.hpp"

namespace camal {
template int act_wgrad_launch<1>(hipStream_t, const ActPlan&, const float*, const ActIn&, float*, ActOut, float*, int, int, int);
}
