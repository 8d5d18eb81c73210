// memory_scan_bf16.hip - the chunked memory kernels for one operand type (compiled side by side with the others).
#include "memory_scan.hpp"

namespace epm {
EPM_SCAN_RUN(bf16)
EPM_SCAN_RUN_PAIR(bf16)
}
