// Attention of trees and within windows over a paged key-value cache: its kernels of bf16 values (attention_blocks.h).
#include "attention_blocks.h"

int mi355::blocks::launch_bf16(BlockParams const &P, bool tree) { return tree ? launch_head<__bf16, true>(P) : launch_head<__bf16, false>(P); }
