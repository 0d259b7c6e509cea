// The tile kernels' work line on the host, against counting one by one: sum_of_halves,
// tile_prefix, and the pieces that units of a share each walk (TileWalk), over random
// ragged batches.  Prints "ok" or the first difference.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "kvm_attend_tile.cuh"

using namespace kvm;

static std::mt19937_64 rng(7);
static int64_t pick(int64_t lo, int64_t hi) { return lo + static_cast<int64_t>(rng() % static_cast<uint64_t>(hi - lo + 1)); }

template <int ROWS, int KEYS>
static bool batch() {
    AttendArgs a{};
    const int n_seq = static_cast<int>(pick(1, 7));
    std::vector<int32_t> start(n_seq + 1), kv(n_seq);
    a.group = static_cast<uint32_t>(pick(1, 12));
    a.n_head_kv = static_cast<uint32_t>(pick(1, 4));
    a.block_tokens = 16;
    a.table_cols = static_cast<uint32_t>(pick(1, 60));
    a.causal = static_cast<uint32_t>(pick(0, 3) != 0);
    for (int s = 0; s < n_seq; ++s) {
        const int64_t n = pick(0, 3) ? pick(0, 400) : pick(0, 3);
        start[s + 1] = start[s] + static_cast<int32_t>(n);
        kv[s] = static_cast<int32_t>(pick(0, 3) ? n + pick(0, 700) : pick(-3, 900));
    }
    a.n_rows = static_cast<uint32_t>(std::max<int64_t>(1, start[n_seq] - pick(0, 1) * pick(0, 20)));
    a.q_start = start.data();
    a.kv_len = kv.data();
    a.n_seq = static_cast<uint32_t>(n_seq);
    a.min_rows = pick(0, 1) ? 1 : 17;
    a.max_rows = 0xffffffffu;

    struct Step { uint32_t seq, head, first; int32_t tile; };
    std::vector<Step> line;              // every (item, key tile) of the call, in order
    for (int s = 0; s < n_seq; ++s) {
        const TileSeq t = tile_seq<ROWS>(a, s);
        int64_t sum = 0;
        for (int64_t i = 0; i <= t.tiles; ++i) {
            if (tile_prefix<ROWS, KEYS>(a, t, i) != sum) return std::printf("prefix of %lld: %lld, not %lld\n", (long long)i, (long long)tile_prefix<ROWS, KEYS>(a, t, i), (long long)sum), false;
            if (i == t.tiles) break;
            // what the tile's rows see, row by row
            int64_t most = 0;
            for (int64_t r = i * ROWS; r < std::min<int64_t>((i + 1) * ROWS, static_cast<int64_t>(t.q.n_new) * a.group); ++r)
                most = std::max<int64_t>(most, attend_limit(a, t.q, static_cast<int32_t>(r / a.group)));
            const int64_t steps = std::max<int64_t>(1, (most + KEYS - 1) / KEYS);
            sum += steps;
            for (uint32_t h = 0; h < a.n_head_kv; ++h)
                for (int64_t k = 0; k < steps; ++k) line.push_back({static_cast<uint32_t>(s), h, static_cast<uint32_t>(i * ROWS), static_cast<int32_t>(k)});
        }
    }
    const uint64_t total = line.size(), units = static_cast<uint64_t>(pick(1, 148));
    const uint64_t share = std::max<uint64_t>(1, (total + units - 1) / units);
    for (uint64_t u = 0; u < units; ++u) {
        uint64_t at = share * u;
        const uint64_t end = std::min(at + share, total);
        if (at >= total) continue;
        TileWalk<ROWS, KEYS> w{};
        w.pos = at;
        w.u1 = end;
        w.share = share;
        uint64_t before = at;
        while (before > 0 && line[before - 1].seq == line[at].seq) --before;
        w.seek(a, line[at].seq, static_cast<int64_t>(at - before));
        TilePiece p;
        while (w.next(a, p)) {
            const uint64_t from = at;
            while (at < end && line[at].seq == p.seq && line[at].head == p.head && line[at].first == p.first) ++at;
            uint64_t last = at;          // the item's end
            while (last < total && line[last].seq == p.seq && line[last].head == p.head && line[last].first == p.first) ++last;
            const bool good = at > from && p.in0 == line[from].tile && p.in1 <= line[at - 1].tile + 1 && p.starts == (line[from].tile == 0) &&
                              p.ends == (last == at) && p.more == (last == at ? 0 : (last - end + share - 1) / share);
            if (!good) return std::printf("piece at %llu of %llu\n", (unsigned long long)from, (unsigned long long)total), false;
        }
        if (at != end) return std::printf("unit ends at %llu, not %llu\n", (unsigned long long)at, (unsigned long long)end), false;
    }
    return true;
}

int main() {
    for (int64_t g = 1; g < 40; ++g)
        for (int64_t e = 0; e < 130; ++e) {
            int64_t sum = 0;
            for (int64_t n = 0; n < 130; ++n) {
                if (sum_of_halves(n, e, g) != sum) return std::printf("sum(%lld, %lld, %lld)\n", (long long)n, (long long)e, (long long)g), 1;
                sum += (2 * n + e) / g;
            }
        }
    for (int i = 0; i < 4000; ++i)
        if (!batch<128, 64>() || !batch<256, 128>()) return 1;
    std::puts("ok");
    return 0;
}
