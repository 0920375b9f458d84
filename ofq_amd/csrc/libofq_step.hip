// Second translation unit of libofq_hip.so: the operators at the two ends of a training step.
#include <algorithm>
#include "common.h"
#include "gemm16.h"
#include "linear_ce.hip"
#include "newton_schulz.hip"
