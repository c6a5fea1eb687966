#include "decay.h"
namespace flare {
bool decay_tc_supported(const DecayArgs&, int) { return false; }
int decay_tc_segments(int, int, int, int, int, int) { return 1; }
int decay_tc(const DecayArgs&, int, cudaStream_t) { return FLARE_EUNSUPPORTED; }
}
