// A row's cut by division (mako_amd/csrc/k_step_cut.hip), a workgroup on the CPU: rows with more tokens in one bin than a list
// holds, and the mass that is looked for at that bin's end, to the last bit; and more mass than there is.
#include "../../mako_amd/csrc/k_step_scan.hip"

#include "../../mako_amd/csrc/k_step_cut.hip"

#include <algorithm>
#include <random>

namespace mako {
namespace step {
namespace {
alignas(16) thread_local unsigned char dyn[sizeof(RowLds)];
}
} // namespace step
} // namespace mako

using namespace mako::step;

namespace {

int failures = 0;

struct Crowded {
    std::vector<float> x;
    mako_cut_desc d{};
    double scale, total;
    uint32_t tokens;

    // 3000 tokens of N(0, 1), 8000 close together below them, 3000 further down
    explicit Crowded(uint32_t seed)
    {
        std::mt19937 rng(seed);
        std::normal_distribution<float> normal;
        for (int i = 0; i < 3000; ++i)
            x.push_back(normal(rng));
        for (int i = 0; i < 8000; ++i)
            x.push_back(-3.0f - 1e-6f * fabsf(normal(rng)));
        for (int i = 0; i < 3000; ++i)
            x.push_back(-4.0f - fabsf(normal(rng)));
        std::shuffle(x.begin(), x.end(), rng);
        tokens = (uint32_t)x.size();
        d.logits = x.data();
        d.n_vocab = tokens;
        d.n_rows = 1;
        d.logits_stride = tokens;
        scale = weight_scale(1.0f);
        total = 0.0;
        for (float v : x)
            total += weight(v, (double)largest(), scale);
    }
    float largest() const { return *std::max_element(x.begin(), x.end()); }

    Cut divide(const Want& want) const
    {
        Cut found = {};
        lanes::run(kThreads, [&] {
            RowLds& lds = *reinterpret_cast<RowLds*>(dyn);
            Row<F32> row(d, 0, largest(), scale);
            const Cut cut = cut_by_division(row, want, total, tokens, lds);
            if (threadIdx.x == 0)
                found = cut;
        });
        return found;
    }
};

void expect(const char* what, uint32_t seed, const Cut& got, uint32_t n, float x)
{
    if (got.n != n || got.x != x) {
        printf("%s, seed %u: %u tokens down to %.9g, expected %u down to %.9g\n", what, seed, got.n, (double)got.x, n, (double)x);
        ++failures;
    }
}

} // namespace

int main()
{
    uint32_t at_the_end = 0;
    for (uint32_t seed = 0; seed < 400 && at_the_end < 6; ++seed) {
        const Crowded g(seed);
        Row<F32> row(g.d, 0, g.largest(), g.scale);
        row.set_unit(g.total);
        const Bins bins(row.max, range_of(g.tokens, g.total, g.scale));
        // units of the tokens before the crowd's bin, and in it
        const uint32_t crowd = bins.of(-3.0f);
        uint64_t before = 0, in = 0;
        uint32_t n = 0, n_in = 0;
        float last = INFINITY;
        for (float v : g.x) {
            const uint32_t bin = bins.of(v);
            const uint64_t units = row.units(row.weigh(v));
            before += bin < crowd ? units : 0;
            n += bin <= crowd;
            if (bin == crowd) {
                in += units;
                ++n_in;
                last = fminf(last, v);
            }
        }
        if (n_in <= kList) {
            printf("no crowd\n");
            return 1;
        }
        // (where the two parts, each rounded, give less than the whole, rounded once)
        const Want want = {0, row.mass(before + in)};
        if (row.mass(before) + row.mass(in) >= want.mass)
            continue;
        lanes::backwards = ++at_the_end % 2 == 0;
        expect("mass at a bin's end", seed, g.divide(want), n, last);
    }
    if (at_the_end < 6) {
        printf("%u rows only\n", at_the_end);
        ++failures;
    }
    const Crowded g(7);
    // (any rank, for comparison: the definition)
    std::vector<float> sorted(g.x);
    std::sort(sorted.begin(), sorted.end(), [](float a, float b) { return a > b; });
    for (uint32_t rank : {1u, 2999u, 3000u, 7000u, 11000u, 11001u, 13999u})
        expect("rank", 7, g.divide(Want{rank, 0.0}), rank, sorted[rank - 1]);
    const Cut all = g.divide(Want{0, g.total * 1.001});
    if (all.n != g.tokens || fabs(all.mass / g.total - 1.0) > 1e-12) {
        printf("more than there is: %u tokens of %g\n", all.n, all.mass);
        ++failures;
    }
    if (!failures)
        printf("ok\n");
    return failures ? 1 : 0;
}
