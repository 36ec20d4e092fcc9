// Bookkeeping of libnd_block.so: last-error string (thread-local) and build id.
#include "blk_common.h"

namespace ndb {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
}

}  // namespace ndb

#ifndef NDB_SRC_HASH
#define NDB_SRC_HASH "unhashed"
#endif
extern "C" const char* nd_block_build_id(void) { return NDB_SRC_HASH; }

extern "C" const char* nd_block_last_error(void) { return ndb::g_err; }
