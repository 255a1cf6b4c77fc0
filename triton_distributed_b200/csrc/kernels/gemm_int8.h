// Products of 8-bit integers: what the launcher in gemm_int8_sm100.cu needs of the few-row kernel (gemm_int8_skinny_sm100.cu).
#pragma once
#include "../include/tdist.h"
#include "gemm_skinny.h"

namespace tdist_host {

// True when the few-row kernel is expected to finish before `other_s` seconds; fills the plan. Looks at sizes only.
bool int8_skinny_plan(int m, int n, int k, double other_s, SkinnyPlan* plan);
int int8_skinny_run(const TdistGemmInt8Args* a, const SkinnyPlan& plan);

}  // namespace tdist_host
