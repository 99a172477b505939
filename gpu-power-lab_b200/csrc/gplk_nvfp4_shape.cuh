// gplk_nvfp4_shape.cuh - the shapes of the few-token NVFP4 kernels' blocks: rings,
// shared memory and TMEM, worked out on the host. Plain C++ without CUDA, so that a
// test can go through every size.
#pragma once

#include <cstddef>
#include <cstdint>

namespace gplk {
namespace fewtok {

constexpr int kMaxTokens = 32;
constexpr int kMaxEntryTokens = 12;             // tokens of one expert that a block takes
constexpr int kMaxPlanes = 7;                   // digit planes of an activation, see gplk_nvfp4_stream.cu
constexpr int kTileRows = 128;
constexpr int kStageK = 256;                    // elements of K per slot
constexpr uint32_t kWBytes = kTileRows * 128;   // codes of a weights' slot
constexpr uint32_t kSfaBytes = 4 * 512;         // its scales
constexpr uint32_t kWSlot = kWBytes + kSfaBytes;
constexpr int kMaxSlots = 10;

// Rings and TMEM of a block. Shared memory: the weights' slots (codes, scales),
// then the activations' (B rows, B scales). TMEM: an accumulator per tile, the
// weights' scale columns per slot, the activations'. Worked out by the host: a
// division takes the device as long as a stage's MMA.
struct Geometry {
    int nb;              // accumulator columns, one per token and plane, padded to 8
    int w_slots, b_slots;
    uint32_t sfb_step;   // bytes from one 64-element block of B scales to the next
    uint32_t image;      // bytes of B rows and scales
    uint32_t b_slot;     // the same, padded to 1 KiB
    uint32_t acc_cols;   // from one accumulator to the next
    uint32_t sfb_cols;   // TMEM columns of a slot's B scales
};

// A slot of activations has no barriers of its own. Tile j of the stream (tile h
// of stage i: j = i * tiles + h) takes weights' slot j % w, so whoever has seen
// that slot free knows that tiles up to j - w are done. Blocks that convert
// fill the activations' slot of stage i then, which has to be free too: b = w
// slots for single tiles, b = w / 2 + 1 for pairs. An Image block copies stage
// i - w + b's then: its activations come out of L2, sooner than the weights, so
// that it holds four stages of them and the more of weights. (With as many slots
// of both, us: 28 x 8192 x 8192 17.1 instead of 16.9, 8 x 16384 x 8192 17.9 and 32 x
// 16384 x 16384 40 as with four.)
constexpr int kImageSlots = 4;

static uint32_t ring_of(const Geometry& g) {
    return (uint32_t)g.w_slots * kWSlot + (uint32_t)g.b_slots * g.b_slot;
}
static uint32_t columns_of(const Geometry& g, int accs) {
    return (uint32_t)accs * g.acc_cols + (uint32_t)g.w_slots * 16 + (uint32_t)g.b_slots * g.sfb_cols;
}

enum class Fill { Convert, Image };

static Geometry geometry(int planes, int ntok, int tiles, Fill fill, uint32_t ring_bytes, uint32_t tmem_cols,
                         int accs = 1, int most_slots = kMaxSlots) {
    Geometry g;
    g.nb = (planes * ntok + 7) & ~7;
    const bool wide = g.nb > 128;  // a second 128 rows of B scales
    // Four blocks of B scales, one per 64 elements of K: 32 lanes of 16 bytes, the
    // scales of rows r, r + 32, r + 64 and r + 96 (and four more for a second 128
    // rows). With up to 32 rows the blocks lie as close as their rows; what a copy
    // of 512 bytes then takes from the next block is never used.
    g.sfb_step = g.nb <= 32 ? 16u * (uint32_t)g.nb : 512u;
    g.image = (uint32_t)g.nb * 128 + (wide ? 4096u : 3 * g.sfb_step + 512);
    g.b_slot = (g.image + 1023) & ~1023u;
    g.acc_cols = ((uint32_t)g.nb + 15) & ~15u;
    g.sfb_cols = wide ? 32 : 16;
    for (g.w_slots = most_slots; g.w_slots > 1; --g.w_slots) {
        g.b_slots = tiles == 2 ? g.w_slots / 2 + 1
                    : fill == Fill::Image && g.w_slots > kImageSlots ? kImageSlots
                                                                     : g.w_slots;
        if (ring_of(g) <= ring_bytes && columns_of(g, accs * tiles) <= tmem_cols) return g;
    }
    g.b_slots = 1;
    return g;
}

// Tensor map of a stack of weight matrices, `rows` rows of k / 2 bytes each: boxes of
// 128 bytes of a tile's rows. The matrices are a dimension of their own, so that a box
// over a matrix's last rows ends with it (zeros) instead of reading the next matrix,
// which may be an expert that no token chose.
struct WeightMap {
    uint64_t sizes[3], pitches[2];
    uint32_t box[3];
};

static WeightMap weight_map(uint64_t rows, uint64_t matrices, uint64_t k) {
    return {{k / 2, rows, matrices}, {k / 2, rows * (k / 2)}, {128, (uint32_t)kTileRows, 1}};
}

// Shared memory and TMEM of a block.
struct Shape {
    uint32_t ring_bytes;  // shared memory of the two rings
    uint32_t tmem_cols;
    size_t smem;
    int per_sm;
};

// Blocks of a cluster wait for one another, and allocating TMEM waits, without a
// limit, for free columns that lie side by side. So no block may wait there for
// columns of another launch, whose cluster could be waiting for this one. A block
// takes half of an SM's 512 columns or all of them, and at least that share of its
// shared memory (228 KiB, 1 KiB of it reserved for each block). At most two halves
// or one whole are resident then, of whatever launches, and a block that has its
// shared memory finds its columns at once. Kernels of other families that take
// TMEM fill more than half of the shared memory and share no SM with these.
// (Registers leave room for no more than two converting blocks on an SM anyway.)
constexpr size_t share_of_smem(uint32_t tmem_cols) { return (size_t)228 * 1024 * tmem_cols / 512 - 1024; }
constexpr bool leaves_no_half(size_t smem) { return smem > share_of_smem(256); }

static size_t overhead_of(size_t control) { return 1024 + ((control + 127) & ~(size_t)127); }

// A block of `tokens` tokens, or of 1 to `tokens` with a geometry for each, of 1 or
// 2 tiles and of at most `stages` stages, with `control` bytes behind its rings:
// half of an SM, or all of it where half holds fewer than three tiles' slots, with no
// more slots than the stages want.
static Shape block_shape(Geometry* geo, int planes, int tokens, bool each, int tiles, Fill fill, int stages,
                         size_t control) {
    const size_t overhead = overhead_of(control);
    const int want = stages < kMaxSlots ? (stages * tiles < kMaxSlots ? stages * tiles : kMaxSlots) : kMaxSlots;
    Shape s;
    uint32_t ring = 0, cols = 0;
    for (uint32_t most = 256; most <= 512; most *= 2) {
        ring = cols = 0;
        bool enough = true;
        for (int t = each ? 1 : tokens; t <= tokens; ++t) {
            const Geometry g =
                geometry(planes, t, tiles, fill, (uint32_t)(share_of_smem(most) - overhead), most, 1, want);
            enough = enough && columns_of(g, tiles) <= most && g.w_slots >= (want < 3 ? want : 3);
            ring = ring_of(g) > ring ? ring_of(g) : ring;
            cols = columns_of(g, tiles) > cols ? columns_of(g, tiles) : cols;
            geo[each ? t - 1 : 0] = g;
        }
        if (enough) break;
    }
    s.tmem_cols = cols <= 256 && ring + overhead <= share_of_smem(256) ? 256 : 512;
    // The slices' sums lie over the rings.
    const uint32_t sums = (uint32_t)(tiles * tokens * kTileRows * 4);
    s.ring_bytes = ((ring > sums ? ring : sums) + 1023) & ~1023u;
    s.smem = s.ring_bytes + overhead;
    if (s.smem < share_of_smem(s.tmem_cols)) s.smem = share_of_smem(s.tmem_cols);
    s.per_sm = (int)(512 / s.tmem_cols);
    return s;
}

// A resident block of the experts' products, for entries of up to `tokens` tokens: two
// tiles, two sets of accumulators, all of an SM.
static Shape item_shape(Geometry* geo, int planes, int tokens, size_t control) {
    Shape s;
    s.ring_bytes = (uint32_t)((share_of_smem(512) - overhead_of(control)) & ~(size_t)1023);
    s.tmem_cols = 512;
    s.smem = share_of_smem(512);
    s.per_sm = 1;
    geo[0] = geometry(planes, tokens, 2, Fill::Convert, s.ring_bytes, s.tmem_cols, 2);
    return s;
}

}  // namespace fewtok
}  // namespace gplk
