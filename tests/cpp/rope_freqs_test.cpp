// kiln::RopeFreqs with its defaults: the frequencies of the published formulas, as the C ABI gives them for 1 to 32 turns (ramp) and
// 1 to 4 (bands). Exit status 1 if one is off by more than the roundings of pow and log.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <vector>

#include "../../kiln_amd/host/kiln_gpu.hpp"

static int bad = 0;
static void same(const char* name, const kiln::RopeFreqs& f, const std::vector<double>& want, double mscale) {
    double worst = 0;
    for (size_t i = 0; i < want.size(); i++) worst = std::max(worst, std::fabs(f.host()[i] / want[i] - 1));
    std::vector<double> dev(want.size());
    const bool copied = hipMemcpy(dev.data(), f.data(), dev.size() * sizeof(double), hipMemcpyDeviceToHost) == hipSuccess &&
                        std::equal(dev.begin(), dev.end(), f.host());
    printf("%-24s worst relative error %.3g, mscale %.7g\n", name, worst, (double)f.mscale());
    if (!(worst <= 8 * 0x1p-52) || f.mscale() != (float)mscale || !copied) bad = 1;
}

int main() {
    const int rot = 128, n = rot / 2;
    const double theta = 5e5, factor = 8, trained = 8192, two_pi = 6.283185307179586477;
    std::vector<double> f(n), bands(n), wide(n), ramp(n);
    for (int i = 0; i < n; i++) f[i] = std::pow(theta, -2.0 * i / rot);
    auto pair = [&](double turns) { return rot * std::log(trained / (turns * two_pi)) / (2 * std::log(theta)); };
    const double lo = std::max(std::floor(pair(32)), 0.0), hi = std::min(std::ceil(pair(1)), rot - 1.0);
    for (int i = 0; i < n; i++) {
        const double turns = trained * f[i] / two_pi, w = std::clamp((i - lo) / std::max(hi - lo, 0.001), 0.0, 1.0);
        const double k4 = std::clamp((turns - 1) / (4 - 1), 0.0, 1.0), k32 = std::clamp((turns - 1) / (32 - 1), 0.0, 1.0);
        bands[i] = f[i] * k4 + f[i] / factor * (1 - k4);
        wide[i] = f[i] * k32 + f[i] / factor * (1 - k32);
        ramp[i] = f[i] / factor * w + f[i] * (1 - w);
    }
    same("none", kiln::RopeFreqs(rot, theta), f, 1);
    same("ramp", kiln::RopeFreqs(rot, theta, KILN_ROPE_RAMP, factor, trained), ramp, 0.1 * std::log(factor) + 1);
    same("bands", kiln::RopeFreqs(rot, theta, KILN_ROPE_BANDS, factor, trained), bands, 1);
    same("bands, slow given", kiln::RopeFreqs(rot, theta, KILN_ROPE_BANDS, factor, trained, 1.0), bands, 1);
    same("bands, both given", kiln::RopeFreqs(rot, theta, KILN_ROPE_BANDS, factor, trained, 1.0, 32.0), wide, 1);
    return bad;
}
