// The selective scan's kernels for elements of type __bf16.
#include "ssm_scan.h"

SRX_SCAN_INSTANTIATE(__bf16)
