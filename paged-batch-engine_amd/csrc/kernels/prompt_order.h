// In which order a prompt batch's tiles are taken where a workgroup has a whole one:
// those that cost the most first. Header-only and constexpr, so the kernel calls it
// on the device, a sequence a lane, and the host tests check it.
//
// Every tile has to come once, whatever the lengths; the order may be a little off. So
// tiles are counted by a function that need not be exact: for one sequence it never
// rises with the cost, at cost 0 it counts all, and at the search's upper end none.
// FP32 is enough for that (exact counts, in FP64 and integers, take 16 mixed prompts from
// 96 to 98.5 us) if differences of costs are taken in integers and the end lies above the
// largest cost by more than FP32's roundings.
#pragma once
#include <stdint.h>

namespace pbe {

// A sequence's tiles: tile t costs base + (t + 1) / rate, in keys.
struct TileRun {
  int32_t tiles = 0;
  uint32_t base = 0;
  float rate = 0;
};
// base and step in sixteenths of a key, as the kernel's model has them; base a multiple.
constexpr TileRun tile_run(int32_t tiles, int64_t base, int64_t step) {
  return {tiles, (uint32_t)(base / 16), step ? 16.f / (float)step : 0x1p40f};
}

// How many of them cost more than c.
constexpr int32_t tiles_above(const TileRun& r, uint32_t c) {
  if (c <= r.base) return r.tiles;
  const float below = (float)(c - r.base) * r.rate;
  if (!(below < (float)r.tiles)) return 0;
  const int32_t n = (int32_t)below;  // may be one of the two above `tiles` that FP32 takes for it
  return n < r.tiles ? r.tiles - n : 0;
}

// Where the search ends, from the largest cost of a tile in 32nds of what tile_run takes
// (below 2^31): 2^-19 above it and more, and the three roundings of tiles_above 2^-22.
constexpr uint32_t cost_end(int32_t most) { return 2u * (uint32_t)most + ((uint32_t)most >> 18) + 64u; }

// low is passed by more than w tiles of the batch, high by at most w: so the w-th of
// the order is among those that pass low and not high. above(c): how many tiles pass c.
struct CostRange {
  uint32_t low, high;
};
template <typename Above>
constexpr CostRange costs_of(uint32_t end, int64_t w, Above above) {
  CostRange r{0, end};
  for (int i = 0; i < 14; ++i) {
    const uint32_t mid = r.low + (r.high - r.low) / 2;
    const bool few = above(mid) <= w;
    r.high = few ? mid : r.high;
    r.low = few ? r.low : mid;
  }
  return r;
}

}  // namespace pbe
