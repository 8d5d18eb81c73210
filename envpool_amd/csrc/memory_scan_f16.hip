// memory_scan_f16.hip - the chunked memory kernels for one operand type (compiled side by side with the others).
#include "memory_scan.hpp"

namespace epm {
EPM_SCAN_RUN(f16)
EPM_SCAN_RUN_PAIR(f16)
}
