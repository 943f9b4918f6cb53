#define FA_INST_HD 256
#define FA_INST_NSUB 1
#define FA_INST_DUAL false
#define FA_INST_NAME launch_kv8_tile_256_128
#include "kv8_tile_inst.inc"
