#define FA_INST_HD 256
#define FA_INST_CODE FA_CODE_INT8
#define FA_INST_NAME launch_kv8_decode_256_int8
#include "kv8_decode_inst.inc"
