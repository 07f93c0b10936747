// Fault flags of the cache operators (q4rdna_kv.cu), part of q4rdna_take_fault.
#pragma once
#include <cstdint>

// Read and cleared; 0xffffffff when they could not be read.
uint32_t q4kv_take_fault();
