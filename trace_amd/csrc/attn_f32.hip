#include "attn_launch.h"

namespace trace {
template int attn_run<float>(AttnPass, const AttnArgs&, hipStream_t);
}
