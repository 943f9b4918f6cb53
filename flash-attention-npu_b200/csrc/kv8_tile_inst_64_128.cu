#define FA_INST_HD 64
#define FA_INST_NSUB 2
#define FA_INST_DUAL true
#define FA_INST_NAME launch_kv8_tile_64_128
#include "kv8_tile_inst.inc"
