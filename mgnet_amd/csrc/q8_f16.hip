// fp16 instantiation of q8.hip (see h16.h)
#define MGN_F16 1
#include "q8.hip"
