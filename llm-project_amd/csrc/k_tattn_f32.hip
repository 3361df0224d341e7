// k_tattn_f32.hip - attention of several new tokens a request over f32 caches (qdev_tattn.h).
#define QTREE_TYPE QLLAMA_KV_F32
#include "qdev_tattn.h"

int qtree::launch_f32(const char *fn, const TaArgs &a, int tile, hipStream_t stream) { return launch_hd<QTREE_TYPE>(fn, a, tile, stream); }
