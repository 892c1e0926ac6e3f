// The host+device arithmetic of kvattention.cuh as it is compiled, on the host:
// one question a line of standard input, one line of answers.
//   split UNITS N U...   the stretches' begins (N + 1 of them), then the stretch of each U
//   place WORD GRID      the partials that a run's place word stands for
//   cut FIRST COUNT      the place word of a cut run
//   apart A N B M        whether N bytes at A and M bytes at B have none in common
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>

#include "kvattention.cuh"

int main() {
    std::string line, what;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        in >> what;
        unsigned a = 0, b = 0, u = 0;
        in >> a >> b;
        if (what == "split") {
            const hsb::Split s(a, b);
            for (unsigned c = 0; c <= b; ++c) std::printf("%u ", s.begin(c));
            while (in >> u) std::printf("%u ", s.of(u));
            std::printf("\n");
        } else if (what == "place") {
            std::printf("%u\n", hsb::run_partials(a, b));
        } else if (what == "apart") {
            unsigned c = 0, d = 0;
            in >> c >> d;
            const auto at = [](unsigned x) { return reinterpret_cast<const void*>((uintptr_t)x); };
            std::printf("%d\n", hsb::apart(at(a), b, at(c), d) ? 1 : 0);
        } else if (what == "cut") {
            std::printf("%u\n", hsb::cut_run(a, b));
        }
    }
}
