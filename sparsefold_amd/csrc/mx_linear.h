// The product of microscaled operands on large grids (256 x 256 tiles): whether it serves `a` (checked as
// sf_hip_mx_linear_fwd does before it asks), and its launch.
#pragma once

#include "sf_common.h"

bool sf_mx_linear_pp_ok(const sf_mx_linear_args* a);
int sf_mx_linear_pp_launch(const sf_mx_linear_args* a, hipStream_t stream);
// The same of 4-bit operands with waves of 128 x 128: whether it serves what the former serves, and its launch.
bool sf_mx_linear_w4_ok(const sf_mx_linear_args* a);
int sf_mx_linear_w4_launch(const sf_mx_linear_args* a, hipStream_t stream);
