// Shared between the translation units of libfrisk_b200.so; not part of the C ABI.
#pragma once
#include <cstdint>

// Sets the text frisk_b200_last_error() returns on the calling thread.
__attribute__((visibility("hidden"))) void frisk_internal_set_error(const char* text);

// Sets how many SM cycles a wait of the streamed 8-bit rows may take, for the launches that follow, and
// returns the limit before: a test makes the waits run out with 0.
extern "C" int64_t frisk_internal_quant_wait_cycles(int64_t cycles);
