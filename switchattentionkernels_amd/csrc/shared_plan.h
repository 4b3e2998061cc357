// The arithmetic of a decode step behind shared prefixes that says which keys a workgroup
// takes and where its partials lie: for the device, where every workgroup works it out for
// itself, and for the host, which sizes the workspace and the grid (and whose tests hold
// the two against each other).
#pragma once

#include "decode_line.h"

namespace swattn {
namespace {

#define SWATTN_BOTH __host__ __device__ __forceinline__

constexpr int kTileRows = 128;       // query rows of a prefix tile, at most
constexpr int kTileKeys = 64;        // keys that a tile's step takes
constexpr uint32_t kMinPiece = 64;   // keys of a prefix piece, at least (128: B4 14.0 us instead of 13.0)
// What a key of a prefix tile costs, in 16ths of a key of the line.  B64 behind 8192 and 32768
// rows with 20: 49.7 and 136 us, 24: 51.0 and 132, 32: 55.7 and 155; 10: 72 and 174.
constexpr uint32_t kTileCost = 24;
constexpr uint32_t kPairPad = 192;   // a pair's start, in keys

SWATTN_BOTH uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// First of a prefix's `rows` rows that a sequence with `own` rows of its own attends.
SWATTN_BOTH int prefix_start(bool full, int rows, int own, int window) {
  const int before = window > own ? window - own : 0;
  return full || before > rows ? 0 : rows - before;
}

// Tiles of `seqs` sequences, tile_inv being 2^20 / tile_seqs rounded up: below 2^11 by 2^16,
// so exact.
SWATTN_BOTH uint32_t tiles_of(uint32_t seqs, uint32_t tile_seqs, uint32_t tile_inv) {
  return ((seqs + tile_seqs - 1u) * tile_inv) >> 20;
}

// Keys of a prefix piece, at most: equal shares of the whole cost over the target's workgroups
// (target_inv: 2^32 / target, rounded up), and a tile is spread over at most 255 pieces.
// line: positions of the line; positions: keys of all tiles of a KV head.
SWATTN_BOTH uint32_t piece_length(uint32_t line, uint32_t positions, uint32_t hkv, uint32_t target_inv, uint32_t prefix_len) {
  const uint64_t cost = line + (static_cast<uint64_t>(positions) * hkv * kTileCost + 15u) / 16u;
  const uint32_t share = static_cast<uint32_t>((cost * target_inv) >> 32) + 1u;
  const uint32_t by_len = (prefix_len + 254u) / 255u;
  return (larger(larger((share * 16u + kTileCost - 1u) / kTileCost, by_len), kMinPiece) + kTileKeys - 1u) & ~(kTileKeys - 1u);
}

// A tile's keys in equal pieces, whole steps of keys: how many, and of how many keys.
struct Cut {
  uint32_t parts, length;
};
SWATTN_BOTH Cut cut_keys(uint32_t keys, uint32_t length) {
  const uint32_t n = (keys + length - 1u) / length;
  const uint32_t each = ((keys + n - 1u) / n + kTileKeys - 1u) & ~(kTileKeys - 1u);
  return Cut{(keys + each - 1u) / each, each};
}

// Of a group's `here` = tiles * KV heads * parts pieces the one that its workgroup number `at`
// takes.  Pieces of the same keys, a tile's each, go one after the other on one XCD (blocks go to the
// eight in turn), which then reads them once: B64 Hq64/Hkv8 behind 32768 rows 136 -> 133.5 us.
struct PieceOf {
  uint32_t tile, kvh, part;
};
SWATTN_BOTH PieceOf piece_of(uint32_t at, uint32_t here, uint32_t tiles, uint32_t parts) {
  const uint32_t x = at & 7u, rest = here & 7u;
  const uint32_t id = x * (here >> 3) + (x < rest ? x : rest) + (at >> 3);
  const uint32_t keys_of = id / tiles, kvh = keys_of / parts;
  return PieceOf{id - keys_of * tiles, kvh, keys_of - kvh * parts};
}

// Workgroups that the line is planned for, where pieces take the first ones.
SWATTN_BOTH uint32_t line_target(uint32_t target, uint32_t pieces, uint32_t least) {
  return larger(target > pieces ? target - pieces : 0u, least);
}

// The share of a position below 2^31, inv being (2^32 - 1) / share rounded down: the quotient
// is one too low at most.
SWATTN_BOTH uint32_t share_of(uint32_t at, uint32_t share, uint32_t inv) {
  const uint32_t n = static_cast<uint32_t>((static_cast<uint64_t>(at) * inv) >> 32);
  return n + (at - n * share >= share ? 1u : 0u);
}

#undef SWATTN_BOTH

}  // namespace
}  // namespace swattn
