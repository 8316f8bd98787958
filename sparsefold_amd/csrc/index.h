// Index arithmetic that kernels share with their tests, which build this header for the host.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#define SF_INDEX __host__ __device__ __forceinline__

// i / n = (i m) >> s of units i < 2^31, n units a page: s = 31 + ceil(log2 n), m = floor(2^s / n) + 1.
struct PageDiv {
  uint32_t m;
  int s;
};
__host__ __device__ inline PageDiv page_div(uint32_t n) {
  int up = 0;
  while ((1u << up) < n) ++up;
  return PageDiv{(uint32_t)((1ull << (31 + up)) / n + 1), 31 + up};
}
SF_INDEX int page_of(const PageDiv& p, uint32_t unit) { return (int)(((uint64_t)unit * p.m) >> p.s); }

// Tile t of gx rows of gy tiles: bands of BAND rows one after another, a band's tiles column by column.
template <int BAND>
SF_INDEX void banded_tile(int t, int gx, int gy, int& row, int& col) {
  const int band = t / (BAND * gy), q = t - band * BAND * gy;
  const int height = BAND < gx - band * BAND ? BAND : gx - band * BAND;
  col = q / height;
  row = band * BAND + q - col * height;
}

// Workgroup b is assumed to run on XCD b % 8.  One workgroup a tile: workgroup b's of `total`, so that each XCD takes a contiguous range.
SF_INDEX int tile_on_xcd(int b, int total) {
  const int xcd = b & 7, rest = total & 7;
  return xcd * (total >> 3) + (xcd < rest ? xcd : rest) + (b >> 3);
}
// Persistent workgroups, a multiple of 8 of them: workgroup b takes tiles first, first + workgroups / 8, .. below `end`.
struct TileWalk {
  int first, end;
};
SF_INDEX TileWalk tiles_on_xcd(uint32_t b, int total) {
  const int per = (total + 7) >> 3, xcd = b & 7;
  return TileWalk{xcd * per + (int)(b >> 3), total < (xcd + 1) * per ? total : (xcd + 1) * per};
}

// 16-byte slot of piece `piece` of a row of 128 (EIGHT) or 64 bytes: the 16 rows that are read together fall on 16 different slots of
// the banks' 256 bytes.
template <bool EIGHT>
SF_INDEX int tile_slot(int row, int piece) {
  return EIGHT ? piece ^ ((row >> 1) & 7) : piece ^ ((row >> 2) & 3);
}

// First of the 16 scales of group g of a row of `blocks` (16 at least): the last group ends with the row.
SF_INDEX int scales_of_group(int g, int blocks) { return 16 * g < blocks - 16 ? 16 * g : blocks - 16; }
