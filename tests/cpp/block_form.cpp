// Prints the form that the products' rule (csrc/block_plan.h) chooses: arguments are rows, experts (0: one group), outputs and
// multiprocessors, four numbers per product.
#include <cstdio>
#include <cstdlib>

#include "block_plan.h"

int main(int argc, char** argv) {
    const char* const names[] = {"Swap16", "Swap32", "Swap128", "Wide128", "Wide256"};
    for (int i = 1; i + 3 < argc; i += 4)
        std::printf("%s\n", names[int(vf::form_of(std::atoll(argv[i]), std::atoll(argv[i + 1]), std::atoll(argv[i + 2]), std::atoll(argv[i + 3])))]);
    return 0;
}
