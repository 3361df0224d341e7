// k_tattn_i8.hip - attention of several new tokens a request over int8 caches (qdev_tattn.h).
#define QTREE_TYPE QLLAMA_KV_I8
#include "qdev_tattn.h"

int qtree::launch_i8(const char *fn, const TaArgs &a, int tile, hipStream_t stream) { return launch_hd<QTREE_TYPE>(fn, a, tile, stream); }
