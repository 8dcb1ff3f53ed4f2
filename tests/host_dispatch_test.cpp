// The dispatcher of csrc/gemm_config.h told what a call is: argv[1] = plugin directory, argv[2] = autotune cache.  One line
// per question: dt M N K group x_dtype zero_points transform, the pick with and without the cache ("-": none).
#include <cstdio>

#include "../sm120_gemm_b200/csrc/gemm_config.h"

int main(int argc, char **argv)
{
    if (argc < 3) return 1;
    KernelRegistry reg;
    reg.quiet = true;
    AutotuneCache cache;
    cache.quiet = true;
    if (!reg.load_dir(argv[1]) || !cache.load(argv[2])) return 1;
    static const int shapes[][4] = {{3, 1, 28672, 8192}, {3, 16, 28672, 8192}, {3, 9, 28672, 8192}, {3, 16, 8192, 28672}, {3, 16, 4096, 4096}, {3, 17, 28672, 8192},
                                    {3, 128, 28672, 8192}, {3, 4, 4097, 4128}, {3, 12, 4096, 14336}, {0, 128, 4096, 14336}, {0, 8192, 8192, 8192}, {1, 8192, 8192, 8192}, {4, 16, 28672, 8192}};
    for (const auto &s : shapes)
        for (int group : {0, 32, 64, 128})
            for (int x_dtype : {GEMM_X_BF16, GEMM_X_F16})
                for (bool zeros : {false, true})
                    for (bool transform : {false, true}) {
                        GemmCallKind kind;
                        kind.group_size = group;
                        kind.x_dtype = x_dtype;
                        kind.zero_points = zeros;
                        kind.transform = transform;
                        const LoadedKernel *h = heuristic_kernel(reg, s[0], s[1], s[2], s[3], 148, kind), *c = select_kernel(reg, cache, s[0], s[1], s[2], s[3], 1, kind);
                        std::printf("%s %d %d %d %d %d %d %d %s %s\n", sm100::kDtypeNames[s[0]], s[1], s[2], s[3], group, x_dtype, zeros, transform,
                                    h ? h->config.name().c_str() : "-", c ? c->config.name().c_str() : "-");
                    }
    return 0;
}
