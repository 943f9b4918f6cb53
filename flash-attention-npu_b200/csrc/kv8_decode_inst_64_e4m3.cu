#define FA_INST_HD 64
#define FA_INST_CODE FA_CODE_E4M3
#define FA_INST_NAME launch_kv8_decode_64_e4m3
#include "kv8_decode_inst.inc"
