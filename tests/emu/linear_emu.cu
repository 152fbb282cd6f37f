// The index arithmetic of the channel-mixing kernels as functions of the CPU, used only by the CPU test-suite.
#include "../../kerops_b200/csrc/linear_core.cuh"

using namespace kdw;

extern "C" long long emu_lin_out_offset(long long row, int col, int cols) { return lin_out_offset(row, col, cols); }

extern "C" float emu_scaled_sum(int sum, float rs, float cs) { return RowScale(rs).of(sum, cs); }

// Quotients that differ from n / d, with a reciprocal that is `ulps` units of its last place off.
extern "C" long long emu_lin_div_misses(const int* n, const int* d, long long count, int ulps) {
    long long misses = 0;
    for (long long i = 0; i < count; ++i) {
        float r = 1.f / (float)d[i];
        for (int k = 0; k < ulps; ++k) r = nextafterf(r, 2.f);
        for (int k = 0; k > ulps; --k) r = nextafterf(r, 0.f);
        misses += lin_div_by(n[i], d[i], r) != n[i] / d[i];
    }
    return misses;
}

extern "C" int emu_few_channels(long long N, long long groups, int sms) { return few_channels(N, groups, sms); }
