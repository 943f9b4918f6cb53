#define FA_INST_HD 128
#define FA_INST_NSUB 1
#define FA_INST_NAME launch_kv8_tile_128_1
#include "kv8_tile_inst.inc"
