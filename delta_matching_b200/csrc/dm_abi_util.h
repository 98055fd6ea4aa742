// What the translation units of the C-ABI layer share: error messages, address checks, tensor maps (defined in dm_abi.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <initializer_list>

#include "../../include/dm_b200.h"

namespace dm {
namespace abi {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct NamedPtr {
  const void* p;
  const char* name;
};

// Each leaves the message of dm_last_error and returns a DM_ERR_* code.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
int check_address(const void* p, const char* name);
int check_addresses(std::initializer_list<NamedPtr> ptrs);
int check_sm100();
// Map over bytes, 128-byte swizzle; up to four dimensions, innermost first.
int encode_byte_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);

}  // namespace abi
}  // namespace dm

#define DM_TRY(expr)            \
  do {                          \
    int _r = (expr);            \
    if (_r != 0) return _r;     \
  } while (0)
