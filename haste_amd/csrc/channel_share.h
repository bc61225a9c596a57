// How the channels of a group are shared among its workgroups (selective_scan.hip).  No HIP in here: the host checks it by itself.
#pragma once

namespace haste_hip {

struct ChannelRange {
  int first, end;
};

// Channels in fours, whose number differs by one at most from workgroup to workgroup, so that the last one, whose last four may be
// incomplete, is not left with a few channels by itself.  For as many fours as workgroups or more.
struct ChannelShare {
  int channels, each, more;  // `more` workgroups have a four besides their `each`
  constexpr ChannelShare(int channels, int workgroups)
      : channels(channels), each((channels + 3) / 4 / workgroups), more((channels + 3) / 4 % workgroups) {}
  constexpr int first(int workgroup) const { return 4 * (workgroup * each + (workgroup < more ? workgroup : more)); }
  constexpr ChannelRange of(int workgroup) const {
    const int end = first(workgroup + 1);
    return {first(workgroup), end < channels ? end : channels};
  }
};

}  // namespace haste_hip
