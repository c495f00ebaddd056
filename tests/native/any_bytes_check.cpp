// Checks any_bytes.h with the optimiser on: a word read again after half of it was written holds the new half, and
// so on for a scale read after a word was written, through pointers that the compiler knows nothing about.
#include <cstdint>
#include <cstdio>

#include "../../qt_llama.cpp_amd/csrc/any_bytes.h"

using namespace mrml;

__attribute__((noinline)) uint32_t word_again(const uint8_t *w, uint8_t *h, uint16_t x)
{
    const uint32_t before = get32(w);
    put16(h, x);
    return before ^ get32(w);
}

__attribute__((noinline)) uint32_t half_again(const uint8_t *h, uint8_t *w, uint32_t x)
{
    const uint32_t before = get16(h);
    *reinterpret_cast<volatile Any32 *>(w) = x;
    return before ^ get16(h);
}

int main()
{
    alignas(16) uint8_t b[16] = {};
    long bad = 0;
    for (uint32_t i = 1; i < 1000; ++i) {
        *reinterpret_cast<Any32 *>(b + 4) = 0;
        bad += word_again(b + 4, b + 6, (uint16_t)i) != i << 16;
        bad += half_again(b + 6, b + 4, 0) != i;
    }
    std::printf("%ld\n", bad);
    return bad != 0;
}
