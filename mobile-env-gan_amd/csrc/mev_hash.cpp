// mev_hash.cpp -- the hash of the sources the library was built from (mev_source_hash): a unit of
// its own, so that a change to one kernel file does not recompile the others.
#include "mev.h"

#ifndef MEV_SRC_HASH
#define MEV_SRC_HASH "unknown"
#endif

const char* mev_source_hash(void) { return MEV_SRC_HASH; }
