// What the translation units of the C boundary share: every exception becomes the message the
// entry point returns, kept by the library until the next failing call on the same thread.
#pragma once
#include <exception>

namespace arb {
const char *fail(const std::exception &e);
const char *fail(const char *msg);
}  // namespace arb

#define ARB_TRY try {
#define ARB_CATCH                                 \
  return nullptr;                                 \
  }                                               \
  catch (const std::exception &e) { return arb::fail(e); } \
  catch (const char *e) { return arb::fail(e); }       \
  catch (...) { return arb::fail("unknown error"); }
