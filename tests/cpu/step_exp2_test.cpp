// The step's weights (mako_amd/csrc/step_common.h): 2^t against the C library's in 80 bits, whose own error of 2^-63 is nothing
// beside what is looked for.
#include <hip/hip_runtime.h>

#include "../../mako_amd/csrc/step_common.h"

using namespace mako::step;

int main()
{
    const double bound = 1.6e-14; // as stated there
    int failures = 0;
    double worst = 0.0, worst_at = 0.0;
    auto look = [&](double t) {
        const double all[4] = {t, t / 2, t, t};
        double four[4];
        exp2_down<4>(all, four);
        const double one = exp2_down(t), finite = exp2_down<true>(t), error = (double)fabsl((long double)one / exp2l((long double)t) - 1.0L);
        if (one != finite || one != four[0] || one != four[3]) {
            printf("2^%.17g: forms differ\n", t);
            ++failures;
        }
        if (error > worst) {
            worst = error;
            worst_at = t;
        }
    };
    for (int i = 0; i <= 400000; ++i)
        look(-i / 200000.0); // (every place between two whole numbers, their middles among them)
    for (int i = 1; i < 200000; ++i)
        look(-1000.0 * i / 200000.0 - 1e-9 * i);
    if (!(worst <= bound)) {
        printf("2^%.17g: off by %.4g of it\n", worst_at, worst);
        ++failures;
    }
    if (exp2_down(0.0) != 1.0 || exp2_down(-INFINITY) != 0.0 || exp2_down(-1100.0) != 0.0) {
        printf("ends\n");
        ++failures;
    }
    if (!failures)
        printf("ok\n");
    return failures ? 1 : 0;
}
