// The SHA-256 of the library's sources, passed by the build recipe, as the library carries it.
#include "../../include/minikv.h"

#ifndef MINIKV_SOURCE_HASH
#define MINIKV_SOURCE_HASH "unknown"
#endif
// The marker prefix lets the build recipe read the hash from the file without loading it.
static const char kSourceHash[] = "minikv-source-hash:" MINIKV_SOURCE_HASH;

extern "C" const char* minikv_source_hash(void) { return kSourceHash + sizeof("minikv-source-hash:") - 1; }
