// Tile facts of the 8-bit kernels for the host planner.
#include "kv8_api.cuh"
#include "kv8_decode_kernel.cuh"
#include "kv8_tile_kernel.cuh"

namespace fa {

template <class Tr>
static Kv8TileInfo info() { return Kv8TileInfo{Tr::BM, Tr::BN, Tr::NTHREADS, Tr::SMEM_BYTES, Tr::RESIDENT}; }

template <int HD>
static Kv8TileInfo decode_info(int rows) {
  return rows == 8 ? info<Kv8Traits<HD, 1, 1>>() : rows == 16 ? info<Kv8Traits<HD, 1, 2>>() : info<Kv8Traits<HD, 2, 2>>();
}
Kv8TileInfo kv8_decode_info(int hd, int rows) { return hd == 64 ? decode_info<64>(rows) : hd == 128 ? decode_info<128>(rows) : decode_info<256>(rows); }

Kv8TileInfo kv8_tile_info(int hd, int rows) {
  if (hd == 64) return rows == 128 ? info<Kv8TileTraits<64, 2, true>>() : info<Kv8TileTraits<64, 2, false>>();
  if (hd == 128) return rows == 128 ? info<Kv8TileTraits<128, 2, true>>() : info<Kv8TileTraits<128, 2, false>>();
  return info<Kv8TileTraits<256, 1, false>>();
}

}  // namespace fa
