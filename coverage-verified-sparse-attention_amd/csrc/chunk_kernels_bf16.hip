// Chunk attention over bf16 caches.
#define CVSA_CHUNK_F8 false
#include "chunk_kernels.h"
