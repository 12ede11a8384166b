// How the selection (sparse_select.hip) and the attention over listed blocks
// (sparse_attention_kernel.h) are launched: rows of a launch and of a workgroup, its waves
// and LDS, from sizes alone.  Host code without HIP, so that it is tested on the CPU over
// every head_dim, list and table width.
#pragma once

#include <stdint.h>

namespace rllm {

constexpr int64_t MAX_WORKGROUPS = ((int64_t(1) << 32) - 1) / 256;   // of a launch, of 256 threads each

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------

constexpr int64_t SELECT_SLAB = int64_t(1) << 30;    // bytes of scratch of one pair of launches (a row's, where that is more)
constexpr int64_t SELECT_CHUNK_MIN = 16, SELECT_CHUNK_MAX = 512;
constexpr int select_m_tiles(int64_t d) { return d > 128 ? 2 : 4; }   // 16-row tiles of a wave, in a chunk

// bytes of scratch of a row: never fewer for a wider table
inline int64_t select_row_bytes(int64_t hkv, int64_t maxb, int64_t& pitch) {
    pitch = (maxb + SELECT_CHUNK_MAX - 1) / SELECT_CHUNK_MAX * SELECT_CHUNK_MAX;
    return hkv * (pitch * 4 + pitch / SELECT_CHUNK_MIN * 4 + pitch);
}
inline int64_t select_bytes(int64_t num_rows, int64_t row_bytes) {
    const int64_t slab = row_bytes > SELECT_SLAB ? row_bytes : SELECT_SLAB;
    return row_bytes == 0 ? 0 : num_rows <= slab / row_bytes ? num_rows * row_bytes : slab;   // (the product may pass 64 bits)
}

struct SelectPlan {
    int64_t pitch, need, slab;  // keys of a list in scratch; bytes of it; rows of a pair of launches
    int64_t chunk, chunks;      // blocks of a scoring workgroup, and such parts of a table (0: nothing is scored)
    bool tiles;                 // rows are scored in tiles
    int group_log2;             // heads of a group, as a power of two, where they are
};

// tiles of a chunk's rows, up to a row of the call (each sequence's last may be cut short)
inline int64_t select_tiles(int64_t rows, int64_t num_seqs, int64_t d, int group_log2) {
    const int64_t tile = 64 * select_m_tiles(d) >> group_log2;
    return (rows + tile - 1) / tile + num_seqs;
}

inline SelectPlan select_plan(int64_t num_rows, int64_t num_seqs, int64_t hq, int64_t hkv, int64_t d, int64_t maxb, int64_t k,
                              bool chunk) {
    SelectPlan p = {0, 0, num_rows, SELECT_CHUNK_MIN, 0, false, 0};
    const int64_t group = hq / hkv;
    while ((1 << p.group_log2) < group) ++p.group_log2;
    // several rows a sequence, one 16-row operand a group: rows share the bounds that they read
    // (704 rows of 1250-1650 blocks, 32/8 heads, head_dim 128: 58 us, 536 row by row)
    p.tiles = chunk && group <= 16 && num_rows >= 2 * num_seqs;
    p.slab = num_rows < MAX_WORKGROUPS / hkv ? num_rows : MAX_WORKGROUPS / hkv;      // a workgroup a list
    if (maxb <= k) return p;                         // every list is the whole sequence
    const int64_t row_bytes = select_row_bytes(hkv, maxb, p.pitch);
    p.need = select_bytes(num_rows, row_bytes);
    if (p.slab > p.need / row_bytes) p.slab = p.need / row_bytes;
    // Row by row, small chunks keep a block's heads together in time and fill the card
    // with few rows (64 rows of 250-2000 blocks: 16 blocks 72 us, 64 92, 128 109); a tile
    // of rows loads its queries for each chunk (704 rows: 32 blocks 79 us, 64 58, 128 67).
    // Not many more workgroups than it takes.
    auto cut = [&] {
        p.chunk = p.tiles ? 64 : SELECT_CHUNK_MIN;
        while (p.chunk < SELECT_CHUNK_MAX && p.slab * ((maxb + p.chunk - 1) / p.chunk) > 32768) p.chunk *= 2;
        p.chunks = (maxb + p.chunk - 1) / p.chunk;
    };
    cut();
    if (p.tiles && select_tiles(num_rows, num_seqs, d, p.group_log2) > MAX_WORKGROUPS / (hkv * p.chunks)) {
        p.tiles = false;
        cut();
    }
    if (!p.tiles && p.slab > MAX_WORKGROUPS / p.chunks) p.slab = MAX_WORKGROUPS / p.chunks;
    return p;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

constexpr int SA_WIN = 64;      // tokens of a wave's window: 4 groups of 16
constexpr int SA_MAX_SPLITS = 8;
constexpr int SA_MAX_LIST = 4096;       // entries of a workgroup's list
constexpr int SA_ENTRY = 10;            // bytes of LDS of an entry
constexpr int SA_LDS = 160 * 1024 - 256;   // of a CU, beside the kernel's few static words

// two workgroups of four waves a CU up to head_dim 128; past it the registers of a window serve one
constexpr int sa_max_waves(int d) { return d > 128 ? 4 : 8; }
constexpr int sa_group_bytes(int d) { return d * 32 + 32; }     // of 16 tokens in LDS; the rest keeps groups on other banks
constexpr int sa_stage_bytes(int d) { return SA_WIN / 16 * sa_group_bytes(d); }

struct SparseShape {
    int64_t rows, num_seqs, hq, hkv, maxb, k;
    int d, bs_log2;
    bool chunk;                 // query_start_loc is given
};
struct SparsePlan {
    int splits, waves;          // workgroups of a unit; waves of one
    int tile, list;             // rows of a workgroup (1, or 16 / heads of a kv head), and the entries its list has room for
};

constexpr int64_t sparse_units(const SparseShape& s) { return s.rows * s.hkv * ((s.hq / s.hkv + 15) / 16); }
constexpr int64_t sparse_windows(const SparseShape& s) { return ((s.k << s.bs_log2) + SA_WIN - 1) / SA_WIN; }

// Few units: a unit's keys come faster to several CUs than to one, so a unit goes to several.
// 8 kv heads, head_dim 128, in a graph, split and not: 1 row on 64 blocks 10.5 and 14.7 us, 4
// rows 13.4 and 14.9; 1 row on 256 14.8 and 36, 8 rows 26.5 and 38.  Where lists are short the
// joining shows before the 128th unit (8 rows on 64 blocks 16.7 and 15.1, 16 19.0 and 15.2).
constexpr bool sparse_few(const SparseShape& s) { return sparse_units(s) <= 128 && sparse_windows(s) > 2; }

constexpr int sa_padded(int list) { return (list + 3) & ~3; }
// long lists beside the windows of wide heads: fewer waves where the LDS of a CU ends
constexpr int sa_waves_beside(int waves, int d, int list) {
    while (waves * sa_stage_bytes(d) + list * SA_ENTRY > SA_LDS) waves /= 2;
    return waves;
}

// `scratch`: whether few units have some to join parts in; a capture on a stream that has none does without.
inline SparsePlan sparse_plan(const SparseShape& s, bool scratch) {
    SparsePlan p = {1, 4, 1, static_cast<int>(s.k)};
    const int64_t units = sparse_units(s), windows = sparse_windows(s);
    if (sparse_few(s)) {
        if (scratch) {
            int64_t splits = 256 / units < SA_MAX_SPLITS ? 256 / units : SA_MAX_SPLITS;
            if (splits > (windows + 1) / 2) splits = (windows + 1) / 2;
            p.splits = static_cast<int>(splits);
            p.waves = windows <= 2 * splits ? 2 : 4;
        } else {
            p.waves = sa_max_waves(s.d);
        }
    }
    p.waves = sa_waves_beside(p.waves, s.d, p.list = sa_padded(p.list));
    // tiles: in a chunk of several rows a sequence, where heads leave columns free, tiles
    // fill the card (on 64 blocks each, 32/8 heads, head_dim 128, in a graph, by single rows and
    // in tiles: 64 rows 24 and 33 us, 96 35 and 33, 128 42 and 33, the rule's border, 704 198 and
    // 116), the union of the lists fits, and the blocks' bits fit where the windows of the
    // waves go that are left beside it
    const int64_t G = s.hq / s.hkv;
    if (s.chunk && s.rows >= 2 * s.num_seqs && G <= 8 && p.splits == 1) {
        int tile = 16;
        while (tile * G > 16) tile /= 2;
        const int64_t most = tile * s.k < s.maxb ? tile * s.k : s.maxb;
        if (units >= 256 * tile && most <= SA_MAX_LIST) {
            const int list = sa_padded(static_cast<int>(most > s.k ? most : s.k));
            const int waves = sa_waves_beside(4, s.d, list);
            if (4 * ((s.maxb + 1) / 2) <= waves * sa_stage_bytes(s.d)) p = {1, waves, tile, list};
        }
    }
    return p;
}

}  // namespace rllm
