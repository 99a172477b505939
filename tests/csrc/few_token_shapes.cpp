// Prints the shape of every block the few-token NVFP4 kernels can launch, a line each:
//   kind planes tokens tiles stages, tmem_cols smem per_sm ring, w_slots b_slots columns ring_used image nb
#include <cstdio>
#include <initializer_list>

#include "gplk_nvfp4_shape.cuh"

using namespace gplk::fewtok;

static void print(const char* kind, int planes, int tokens, bool each, int tiles, int accs, int stages, const Shape& s, const Geometry* geo) {
    for (int t = each ? 1 : tokens; t <= tokens; ++t) {
        const Geometry& g = geo[each ? t - 1 : 0];
        printf("%s %d %d %d %d %u %zu %d %u %d %d %u %u %u %d\n", kind, planes, t, tiles, stages, s.tmem_cols, s.smem, s.per_sm,
               s.ring_bytes, g.w_slots, g.b_slots, columns_of(g, accs * tiles), ring_of(g), g.image, g.nb);
    }
}

int main() {
    Geometry geo[kMaxTokens];
    for (int planes : {6, 7}) {
        for (size_t control : {(size_t)256, (size_t)1024})
            for (int stages = 1; stages <= 24; ++stages) {
                for (int t = 1; t <= kMaxTokens; ++t)
                    for (Fill fill : {Fill::Convert, Fill::Image})
                        print(fill == Fill::Image ? "image" : "convert", planes, t, false, 1, 1, stages,
                              block_shape(geo, planes, t, false, 1, fill, stages, control), geo);
                for (int t = 1; t <= kMaxEntryTokens; ++t)
                    print("gateup", planes, t, true, 2, 1, stages,
                          block_shape(geo, planes, t, true, 2, Fill::Convert, stages, control), geo);
            }
        for (int t = 1; t <= kMaxEntryTokens; ++t)
            print("item", planes, t, false, 2, 2, 0, item_shape(geo, planes, t, 512), geo);
    }
    return 0;
}
