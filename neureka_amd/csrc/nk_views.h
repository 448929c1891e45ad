// Whether two strided views share an element (host only).
#ifndef NK_VIEWS_H
#define NK_VIEWS_H

#include <algorithm>
#include <cstdint>
#include <numeric>

namespace nk {

struct View {                                               // elements at first + sum of step[k] i[k], 0 <= i[k] < extent[k]
    static constexpr int MOST = 8;
    int64_t first = 0, extent[MOST], step[MOST];
    int rank = 0;
    int64_t least() const { int64_t x = first; for (int k = 0; k < rank; k++) x += std::min<int64_t>(0, step[k] * (extent[k] - 1)); return x; }
    int64_t most() const { int64_t x = first; for (int k = 0; k < rank; k++) x += std::max<int64_t>(0, step[k] * (extent[k] - 1)); return x; }
};

// Is there i, j with  a.first + sum of a.step i  =  b.first + sum of b.step j ?  Every step times its index is a term of one sum that has to come to b - a;
// terms of equal step count as one.  Taken from the largest step down, a term has only the few values that leave what the smaller ones
// reach.  Steps in no proportion could make that a long search: after `tries` it is taken as yes.
inline bool views_meet(const View& a, const View& b, int tries = 20000) {
    if (a.most() < b.least() || b.most() < a.least()) return false;
    struct Term { int64_t step, low, high; } terms[2 * View::MOST];
    int n = 0;
    const auto add = [&](int64_t step, int64_t low, int64_t high) {
        if (step == 0 || low == high) return;
        if (step < 0) { step = -step; std::swap(low, high); low = -low; high = -high; }
        for (int k = 0; k < n; k++) if (terms[k].step == step) { terms[k].low += low; terms[k].high += high; return; }
        terms[n++] = {step, low, high};
    };
    for (int k = 0; k < a.rank; k++) add(a.step[k], 0, a.extent[k] - 1);
    for (int k = 0; k < b.rank; k++) add(b.step[k], 1 - b.extent[k], 0);
    std::sort(terms, terms + n, [](const Term& x, const Term& y) { return x.step > y.step; });
    int64_t least[2 * View::MOST + 1] = {}, most[2 * View::MOST + 1] = {}, divisor[2 * View::MOST + 1] = {};      // what the terms from k on reach
    for (int k = n; k-- > 0;) {
        least[k] = least[k + 1] + terms[k].step * terms[k].low;
        most[k] = most[k + 1] + terms[k].step * terms[k].high;
        divisor[k] = std::gcd(divisor[k + 1], terms[k].step);
    }
    const auto down = [](int64_t x, int64_t by) { return x >= 0 ? x / by : -((-x + by - 1) / by); };     // rounded towards minus infinity
    const auto search = [&](const auto& self, int k, int64_t left) -> bool {
        if (left < least[k] || left > most[k]) return false;
        if (k == n) return true;
        if (left % divisor[k] != 0) return false;
        if (--tries < 0) return true;
        const Term& t = terms[k];
        const int64_t from = std::max(t.low, -down(most[k + 1] - left, t.step)), to = std::min(t.high, down(left - least[k + 1], t.step));
        for (int64_t v = from; v <= to; v++)
            if (self(self, k + 1, left - t.step * v)) return true;
        return false;
    };
    return search(search, 0, b.first - a.first);
}

}  // namespace nk
#endif
