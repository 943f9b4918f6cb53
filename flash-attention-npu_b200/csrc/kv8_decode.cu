// Tile facts of the 8-bit kernels for the host planner.
#include "kv8_api.cuh"
#include "kv8_decode_kernel.cuh"
#include "kv8_tile_kernel.cuh"

namespace fa {

template <class Tr>
static Kv8TileInfo info() { return Kv8TileInfo{Tr::BM, Tr::BN, Tr::NTHREADS, Tr::SMEM_BYTES, Tr::RESIDENT}; }

Kv8TileInfo kv8_decode_info(int hd, bool wide) {
  if (hd == 64) return wide ? info<Kv8Traits<64, 2>>() : info<Kv8Traits<64, 1>>();
  if (hd == 128) return wide ? info<Kv8Traits<128, 2>>() : info<Kv8Traits<128, 1>>();
  return wide ? info<Kv8Traits<256, 2>>() : info<Kv8Traits<256, 1>>();
}

Kv8TileInfo kv8_tile_info(int hd, int subs) {
  if (hd == 64) return subs == 1 ? info<Kv8TileTraits<64, 1>>() : info<Kv8TileTraits<64, 2>>();
  if (hd == 128) return subs == 1 ? info<Kv8TileTraits<128, 1>>() : info<Kv8TileTraits<128, 2>>();
  return info<Kv8TileTraits<256, 1>>();
}

}  // namespace fa
