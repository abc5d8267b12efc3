// Chunk attention over caches of 8 bits.
#define CVSA_CHUNK_F8 true
#include "chunk_kernels.h"
