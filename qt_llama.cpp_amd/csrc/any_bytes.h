// any_bytes.h -- bytes read and written in words of other types (host and device).
//
// Rows of quantised blocks are copied into LDS in words of 2, 4 or 16 bytes and read back as scales (2 bytes) and
// quants (4 or 8 bytes).  Through ordinary uint16_t and uint32_t pointers the compiler may take such a store and such a
// load for independent (they cannot name the same object of the language) and use what it read before the store; these types may
// name any object.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define MRML_AB_HD __host__ __device__ __forceinline__
#else
#define MRML_AB_HD static inline
#endif

namespace mrml {

typedef uint32_t __attribute__((may_alias)) Any32;
typedef uint16_t __attribute__((may_alias)) Any16;
typedef int64_t __attribute__((may_alias)) Any64;
#if defined(__HIPCC__)
typedef uint32_t Any128 __attribute__((ext_vector_type(4), may_alias));
#endif

MRML_AB_HD uint32_t get32(const uint8_t *p) { return *reinterpret_cast<const Any32 *>(p); }
MRML_AB_HD uint16_t get16(const uint8_t *p) { return *reinterpret_cast<const Any16 *>(p); }
MRML_AB_HD void put16(uint8_t *p, uint16_t x) { *reinterpret_cast<Any16 *>(p) = x; }

}  // namespace mrml
