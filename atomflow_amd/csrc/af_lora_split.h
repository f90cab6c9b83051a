// af_lora_split.h — how the adapters' first product cuts K, for the launch, the kernels and the host's tests
// (plain C++).
#pragma once

namespace af {

constexpr int kLoraParts = 8;      // parts of K, at most
constexpr int kLoraPartMin = 512;  // k of a part, at least
constexpr int kLoraPiece = 64;     // k of a piece: what the LDS form loads at a time

// By k alone, so that a token's sums have the same order in every launch. A part is four chains of
// whole pieces; rounding up to them can leave fewer parts than asked for (k 5120: 7 of 768), and
// none is empty.
struct LoraSplit {
    int parts, part_k;
};
constexpr LoraSplit lora_split(int k) {
    const int wanted = (k - 1) / kLoraPartMin + 1;
    const int each = (k - 1) / (wanted < kLoraParts ? wanted : kLoraParts) + 1;
    const int part_k = (each + 255) / 256 * 256;
    return {(k - 1) / part_k + 1, part_k};
}

// K [k0, k1) of a workgroup that takes one of `splits` parts, or all of K (splits 1), in pieces.
struct LoraRange {
    int k0, k1, pieces;
};
constexpr LoraRange lora_range(int k, int part_k, int splits, int split) {
    const int k0 = splits == 1 ? 0 : split * part_k;
    const int k1 = splits == 1 || k0 + part_k > k ? k : k0 + part_k;
    return {k0, k1, (k1 - k0 + kLoraPiece - 1) / kLoraPiece};
}

// What is added to where the last piece's loads of 8 elements start (8 * eighth behind the piece's):
// past K they repeat the row's last 8.
constexpr int lora_pull_back(int k, const LoraRange& r, int eighth) {
    const int past = k - 8 - (r.k0 + kLoraPiece * (r.pieces - 1) + 8 * eighth);
    return past < 0 ? past : 0;
}

}  // namespace af
