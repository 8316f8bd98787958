// The product of microscaled operands on large grids (256 x 256 tiles): whether it serves `a` (checked as
// sf_hip_mx_linear_fwd does before it asks), and its launch.
#pragma once

#include "sf_common.h"

bool sf_mx_linear_pp_ok(const sf_mx_linear_args* a);
int sf_mx_linear_pp_launch(const sf_mx_linear_args* a, hipStream_t stream);
