// Host run of the reports that threads get of kernels that have given up (reports.h).  Test code only.
#include <thread>

#include "../../openfish_b200/csrc/reports.h"

static Reports reports;
static thread_local int known[Reports::kDevices];

extern "C" void begin(int device) { reports.begin(device, known); }
extern "C" int take(int device, int count) { return reports.take(device, known, count); }
