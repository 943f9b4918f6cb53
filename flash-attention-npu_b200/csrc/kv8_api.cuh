// Interface between the host planner of the 8-bit KV cache and its kernels.
#pragma once

#include "kv8.cuh"

namespace fa {

struct Kv8TileInfo {
  int block_m, block_n, threads, smem_bytes, resident;
};
// Decode kernel: `hd` tile width (64, 128, 256), tiles of 8, 16 or 32 rows.
Kv8TileInfo kv8_decode_info(int hd, int rows);
#define FA_KV8_LAUNCHER(NAME_) \
  cudaError_t NAME_(int rows, const Kv8Params& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, int grid, cudaStream_t st);
FA_KV8_LAUNCHER(launch_kv8_decode_64_e4m3)
FA_KV8_LAUNCHER(launch_kv8_decode_64_int8)
FA_KV8_LAUNCHER(launch_kv8_decode_128_e4m3)
FA_KV8_LAUNCHER(launch_kv8_decode_128_int8)
FA_KV8_LAUNCHER(launch_kv8_decode_256_e4m3)
FA_KV8_LAUNCHER(launch_kv8_decode_256_int8)
#undef FA_KV8_LAUNCHER

// Tile kernel: tiles of 128 or (up to 128 columns) 256 rows.
Kv8TileInfo kv8_tile_info(int hd, int rows);
cudaError_t launch_kv8_tile_64_128(const Kv8Params& p, int grid, cudaStream_t st);
cudaError_t launch_kv8_tile_64_256(const Kv8Params& p, int grid, cudaStream_t st);
cudaError_t launch_kv8_tile_128_128(const Kv8Params& p, int grid, cudaStream_t st);
cudaError_t launch_kv8_tile_128_256(const Kv8Params& p, int grid, cudaStream_t st);
cudaError_t launch_kv8_tile_256_128(const Kv8Params& p, int grid, cudaStream_t st);

cudaError_t launch_kv8_append(const fa_kv8_append_params& p, int num_sm, int32_t* status, cudaStream_t st);
cudaError_t launch_kv8_append_dense(const Kv8Params& p, cudaStream_t st);
cudaError_t launch_kvcache_plan(const fa_kvcache_plan_params& p, int num_sm, int32_t* status, cudaStream_t st);

}  // namespace fa
