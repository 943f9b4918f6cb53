#define FA_INST_HD 64
#define FA_INST_NSUB 1
#define FA_INST_NAME launch_kv8_tile_64_1
#include "kv8_tile_inst.inc"
