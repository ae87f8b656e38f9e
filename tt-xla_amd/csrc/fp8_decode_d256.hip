// Decode attention over the 8-bit cache, head size 256.
#include "fp8_decode_kernel.h"

namespace ttpa {
namespace decode {

bool launch_fp8_d256(const void *args, hipStream_t st) { return launch_fp8<256>(*static_cast<const Fp8Args *>(args), st); }

}  // namespace decode
}  // namespace ttpa
