// Host helpers shared by the translation units that launch kernels.
#ifndef CVCUDA_B200_HOST_COMMON_H
#define CVCUDA_B200_HOST_COMMON_H

namespace b200pp {

// Keeps the message for b200ppGetLastErrorMessage() and returns `status`.
int fail(int status, const char *fmt, ...);

// After a launch: reports a failed one, counts a good one.
int check_launch(const char *what);

} // namespace b200pp

#endif
