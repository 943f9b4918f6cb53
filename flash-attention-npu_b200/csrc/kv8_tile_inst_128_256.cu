#define FA_INST_HD 128
#define FA_INST_NSUB 2
#define FA_INST_DUAL false
#define FA_INST_NAME launch_kv8_tile_128_256
#include "kv8_tile_inst.inc"
