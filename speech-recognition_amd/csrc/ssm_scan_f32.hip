// The selective scan's kernels for elements of type float.
#include "ssm_scan.h"

SRX_SCAN_INSTANTIATE(float)
