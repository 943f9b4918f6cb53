#define FA_INST_HD 256
#define FA_INST_NAME launch_kv8_tile_256
#include "kv8_tile_inst.inc"
