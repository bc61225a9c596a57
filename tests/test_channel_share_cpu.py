"""How a group's channels are shared among the workgroups of a scan (haste_amd/csrc/channel_share.h), on the host."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "haste_amd/csrc/channel_share.h"
// fewest and most channels of a workgroup; -1 where the ranges do not follow one another in fours from 0 to `channels`
extern "C" int spread(int channels, int workgroups, int* fewest, int* most) {
  int at = 0;
  *fewest = channels;
  *most = 0;
  for (int i = 0; i < workgroups; ++i) {
    const haste_hip::ChannelRange r = haste_hip::ChannelShare(channels, workgroups).of(i);
    if (r.first != at || r.first % 4 != 0 || r.end <= r.first) return -1;
    at = r.end;
    if (r.end - r.first < *fewest) *fewest = r.end - r.first;
    if (r.end - r.first > *most) *most = r.end - r.first;
  }
  return at == channels ? 0 : -1;
}
"""


@pytest.fixture(scope="module")
def spread(tmp_path_factory):
    at = tmp_path_factory.mktemp("channel_share")
    (at / "spread.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + ROOT, str(at / "spread.cpp"), "-o", str(at / "spread.so")],
                   check=True, timeout=60)
    return ctypes.CDLL(str(at / "spread.so")).spread


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_no_workgroup_is_left_with_a_few_channels(spread, block):
    """block: the channels that a workgroup has room for."""
    fewest, most = ctypes.c_int(), ctypes.c_int()
    for channels in [*range(1, 5000), 65535, 65537, 10 ** 6 + 1, 2 ** 30 // 66]:
        workgroups = -(-channels // block)
        assert spread(channels, workgroups, ctypes.byref(fewest), ctypes.byref(most)) == 0, channels
        assert most.value <= block and most.value - fewest.value <= 7, channels  # a four less, and an incomplete one
        if workgroups > 1:
            assert fewest.value >= block // 4, channels


def test_channels_that_used_to_leave_one(spread):
    fewest, most = ctypes.c_int(), ctypes.c_int()
    for channels, block, least in ((961, 64, 57), (1025, 64, 57), (1026, 64, 58), (2049, 64, 57), (4097, 64, 57), (129, 16, 9)):
        assert spread(channels, -(-channels // block), ctypes.byref(fewest), ctypes.byref(most)) == 0
        assert fewest.value >= least, (channels, fewest.value)
