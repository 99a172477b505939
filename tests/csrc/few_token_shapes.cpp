// Prints, a line each, for stacks of weight matrices
//   map rows matrices k, bytes of other matrices that a matrix's boxes cover, bytes of its own
// and the shape of every block the few-token NVFP4 kernels can launch:
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

// Bytes of other matrices that the boxes over matrix e of a stack cover, as the kernels place them.
static void print_map(uint64_t rows, uint64_t matrices, uint64_t k) {
    const WeightMap m = weight_map(rows, matrices, k);
    uint64_t outside = 0, covered = 0;
    for (uint64_t e = 0; e < matrices; ++e)
        for (uint64_t tile = 0; tile * kTileRows < rows; ++tile)
            for (uint64_t x = 0; x < k / 2; x += 128)
                for (uint64_t r = tile * kTileRows; r < tile * kTileRows + m.box[1] && r < m.sizes[1]; ++r)
                    for (uint64_t z = e; z < e + m.box[2] && z < m.sizes[2]; ++z)
                        for (uint64_t c = x; c < x + m.box[0] && c < m.sizes[0]; c += 16) {
                            const uint64_t at = c + r * m.pitches[0] + z * m.pitches[1];
                            const uint64_t matrix = rows * (k / 2);
                            (at >= e * matrix && at < (e + 1) * matrix ? covered : outside) += 16;
                        }
    printf("map %llu %llu %llu %llu %llu\n", (unsigned long long)rows, (unsigned long long)matrices,
           (unsigned long long)k, (unsigned long long)outside, (unsigned long long)covered);
}

int main() {
    for (uint64_t rows : {(uint64_t)64, (uint64_t)128, (uint64_t)192, (uint64_t)704, (uint64_t)1000})
        for (uint64_t k : {(uint64_t)64, (uint64_t)320, (uint64_t)1088}) print_map(rows, 3, k);
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
