/* A stand-in for a library call that lasts until another thread sets `flag` (0), at most five seconds (1). */
#include <time.h>

volatile int entered = 0, flag = 0;

int wait_for_flag(void) {
  const struct timespec ms = {0, 1000000};
  entered = 1;
  for (int i = 0; i < 5000 && !flag; ++i) nanosleep(&ms, 0);
  return flag ? 0 : 1;
}

const char* no_flag(void) { return "no other thread ran during the call"; }
