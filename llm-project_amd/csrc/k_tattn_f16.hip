// k_tattn_f16.hip - attention of several new tokens a request over f16 caches (qdev_tattn.h).
#define QTREE_TYPE QLLAMA_KV_F16
#include "qdev_tattn.h"

int qtree::launch_f16(const char *fn, const TaArgs &a, int tile, hipStream_t stream) { return launch_hd<QTREE_TYPE>(fn, a, tile, stream); }
