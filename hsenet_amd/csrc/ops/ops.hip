// what the operators' library says about itself (hs_ops_build_id is compiled in by build.py)
#include "../../../include/hsenet_ops.h"
extern "C" int hs_ops_version(void) { return HS_OPS_ABI_VERSION; }
