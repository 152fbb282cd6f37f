// The index arithmetic of the channel-mixing kernels as functions of the CPU, used only by the CPU test-suite.
#include "../../kerops_b200/csrc/linear_core.cuh"

using namespace kdw;

extern "C" long long emu_lin_out_offset(long long row, int col, int cols) { return lin_out_offset(row, col, cols); }

extern "C" float emu_scaled_sum(int sum, float rs, float cs) { return RowScale(rs).of(sum, cs); }
