// The chunk attention's host side of positions and tiles, for tests without a GPU.
#include "../../insitu_b200/csrc/chunk_tiles.cuh"

int ins::fail(int code, const std::string &) { return code; }

using namespace ins;

extern "C" {

// Checks one sequence of `len` tokens, the last n of them new, in every row tile
// against the definition; 0, or the number of the rule that is broken.
int chunk_check(int window, int sinks, int len, int n, int groups) {
    const ChunkView v{window, sinks};
    ChunkSeq s = walk_of(v, 0, len, n, 0);
    const int span = v.span(s);
    if (s.early % WALK || s.skip % WALK || s.early < 0 || s.skip < 0 || span < 1 || span > len) return 1;
    auto sees = [&](int p, int t) { return t <= p && (t > p - window || t < sinks); };
    // the walk holds every position that a new token sees, each once, in order
    std::vector<char> walked((size_t)len, 0);
    for (int i = 0, last = -1; i < span; ++i) {
        const int p = v.at(s, i);
        if (p <= last || p >= len) return 2;
        walked[(size_t)p] = 1;
        last = p;
    }
    const int per = TL_ROWS / groups;
    s.rts = (n + per - 1) / per;
    for (int rt = 0; rt < s.rts; ++rt) {
        const RowTile t = row_tile(v, s, groups, rt);
        if (t.n < 1 || t.first != rt * per || t.n > per || t.first + t.n > n || t.tiles < 1) return 3;
        const int p_lo = s.context + t.first, p_hi = p_lo + t.n - 1;
        const WholeTiles whole = whole_tiles(v, p_lo, p_hi, t.early, t.jump);
        std::vector<char> tiles((size_t)(len + TL_TILE - 1) / TL_TILE, 0);
        for (int j = 0; j < t.tiles; ++j) {
            const int tile = j < t.early ? j : j + t.jump;
            if (tile < 0 || tile >= (int)tiles.size() || tiles[(size_t)tile]) return 4;
            tiles[(size_t)tile] = 1;
            // its image is the walk's tile of these positions
            const int walk = tile < s.early / TL_TILE ? tile : tile - s.skip / TL_TILE;
            if (walk < 0 || walk * TL_TILE >= span || v.at(s, walk * TL_TILE) != tile * TL_TILE) return 5;
            bool all = true;
            for (int x = 0; x < TL_TILE; ++x)
                for (int p : {p_lo, (p_lo + p_hi) / 2, p_hi}) all &= sees(p, tile * TL_TILE + x);
            if (whole(j) && !all) return 6;
        }
        for (int p = p_lo; p <= p_hi; p += std::max(1, t.n / 3)) {
            const ChunkView::Row row = v.row(s, p - s.context);
            for (int at = 0; at < len; ++at) {
                if (sees(p, at) && (!walked[(size_t)at] || !tiles[(size_t)(at / TL_TILE)])) return 7;
                if (row.sees(at) != sees(p, at)) return 8;
                if (at % 16 == 0) {
                    const uint32_t bits = row.bits(at);
                    for (int k = 0; k < 32; ++k)
                        if ((bits >> k & 1u) != (uint32_t)sees(p, at + k)) return 9;
                }
            }
        }
    }
    // tiles of the short kernels that need no mask
    for (int i = 0; i + FEW_TILE <= span; i += FEW_TILE)
        if (v.whole(s, v.at(s, i), FEW_TILE))
            for (int x = 0; x < FEW_TILE; ++x)
                for (int p : {s.context, len - 1})
                    if (!sees(p, v.at(s, i) + x)) return 10;
    return 0;
}

}  // extern "C"
