// Host build of attend_rows_plan.hpp: the byte order of an 8-bit KV state is
// one to one and inside its record, and every plan covers its rows and keys
// with scratch inside the bound that callers size by.
#include "attend_rows_plan.hpp"
#include "check.hpp"

#include <cstdint>
#include <algorithm>
#include <cmath>
#include <random>
#include <vector>

int main() {
    for (uint32_t hd = 2; hd <= 256; hd += 2) {
        const syn::kv8_shape s = syn::kv8_shape_of(1000, 3, hd);
        CHECK(s.hdp % 32 == 0 && s.hdp >= hd && s.hdp < hd + 32 && s.tiles == 16);
        CHECK(s.tile_bytes % 16 == 0 && s.v_at == 64 * s.hdp && s.ks_at == 2 * s.v_at);
        std::vector<int> k(s.v_at, 0), v(s.v_at, 0);
        for (uint32_t key = 0; key < 64; ++key) {
            for (uint32_t d = 0; d < s.hdp; ++d) {
                const uint32_t a = syn::kv8_k_at(s.hdp, key, d), b = syn::kv8_v_at(key, d);
                CHECK(a < s.v_at && b < s.v_at);
                ++k[a];
                ++v[b];
                // Four dims of K and four keys of V share an aligned word.
                CHECK(d % 4 == 0 || a == syn::kv8_k_at(s.hdp, key, d - 1) + 1);
                CHECK(key % 4 == 0 || b == syn::kv8_v_at(key - 1, d) + 1);
            }
        }
        for (uint32_t i = 0; i < s.v_at; ++i) {
            CHECK(k[i] == 1 && v[i] == 1);
        }
    }

    std::mt19937 r(7);
    const auto upto = [&](uint32_t most) {
        const double x = std::uniform_real_distribution<>(0.0, 1.0)(r);
        return static_cast<uint32_t>(std::max(1.0, std::pow(double(most), x)));
    };
    for (int i = 0; i < 3000; ++i) {
        const uint32_t group = upto(40), n_kv = upto(64), hd = 2 * upto(128), max_ctx = upto(300000);
        const uint32_t n = upto(max_ctx), max_n = n + upto(100) - 1;
        const uint32_t len = n + (max_ctx > n ? static_cast<uint32_t>(r()) % (max_ctx - n + 1) : 0);
        const bool by_pairs = i % 3 == 0, halves = by_pairs || i % 3 == 1;
        const syn::attend_plan p = syn::plan_attend_rows(n, group, n_kv, hd, len, halves, by_pairs);
        CHECK(!by_pairs || p.kernel <= syn::attend_many16);
        CHECK(p.kernel != syn::attend_turns || hd <= 128);
        CHECK(p.kernel != syn::attend_few || p.row_blocks == 1);
        CHECK(p.kernel != syn::attend_few || !halves || hd <= 192);
        CHECK(uint64_t{p.row_blocks} * p.block_rows >= uint64_t{n} * group);
        CHECK(uint64_t{p.row_blocks - 1} * p.block_rows < uint64_t{n} * group);
        const uint32_t tiles = (len + 63) / 64;
        CHECK(uint64_t{p.chunk} * p.splits >= tiles && uint64_t{p.chunk} * (p.splits - 1) < tiles);
        CHECK(p.splits >= 1 && p.splits <= syn::attend_max_splits);
        CHECK(syn::attend_scratch_floats(p, n_kv, uint64_t{n} * group, hd) <=
              syn::attend_scratch_bound(std::min(max_n, max_ctx), group, n_kv, hd, max_ctx, halves, by_pairs));
    }
    CHECK_DONE();
}
