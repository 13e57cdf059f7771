// The selective scan's kernels for elements of type _Float16.
#include "ssm_scan.h"

SRX_SCAN_INSTANTIATE(_Float16)
