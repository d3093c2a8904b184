#include "attn_launch.h"

namespace trace {
template int attn_run<__bf16>(AttnPass, const AttnArgs&, hipStream_t);
}
