#include "attn_launch.h"

namespace trace {
template int attn_run<_Float16>(AttnPass, const AttnArgs&, hipStream_t);
}
