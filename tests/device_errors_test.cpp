// take_device_errors with the device's words in a fake: every combination of errors, each followed by a second look.
#include <cstdio>

#include "../flint_mac_b200/csrc/device_errors.h"

struct Fake {
    int prefill = 0, decode = 0, exchange = 0, counters = 3;
    static int take(int &w) {
        const int v = w;
        w = 0;
        return v;
    }
    int take_prefill() { return take(prefill); }
    int take_decode() { return take(decode); }
    int take_exchange() { return take(exchange); }
    void clear_counters() { counters = 0; }
};

int main() {
    int wrong = 0;
    for (int bits = 0; bits < 8; bits++) {
        Fake f;
        f.prefill = bits & 1 ? 1 : 0;
        f.decode = bits & 2 ? 4 : 0;
        f.exchange = bits & 4 ? 7 : 0;
        const std::string s = flint::take_device_errors(f);
        const bool said = ((s.find("prefill kernel reported device error 1") != s.npos) == bool(bits & 1)) &&
                          ((s.find("decode kernel reported device error 4") != s.npos) == bool(bits & 2)) &&
                          ((s.find("ran out (exchange error 7)") != s.npos) == bool(bits & 4)) && (s.empty() == (bits == 0));
        const bool clear = !f.prefill && !f.decode && !f.exchange && f.counters == (bits & 2 ? 0 : 3);
        if (!said || !clear || !flint::take_device_errors(f).empty()) {
            std::printf("errors %d: '%s', counters %d\n", bits, s.c_str(), f.counters);
            wrong++;
        }
    }
    if (!wrong) std::printf("device errors ok\n");
    return wrong != 0;
}
