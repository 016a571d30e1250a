"""How a layer's tiles are cut along the sum (npa_amd/csrc/turns.hpp), built for
the host: whatever the offsets hold, the slices' places stay inside the workspace
that the library asks for."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

import npa_amd
from npa_amd.sphops import _native

lib = _native.lib
CSRC = os.path.join(os.path.dirname(npa_amd.__file__), "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
SOURCE = """
#include "turns.hpp"
extern "C" int64_t tiles_of(const int32_t* offsets, int experts, int64_t slots, int64_t size) {
  int64_t n = 0;
  for (int e = 0; e <= experts; ++e) {
    const sphops::GroupRows g = sphops::group_rows(offsets, experts, slots, e);
    if (g.lo < 0 || g.lo > g.hi || g.hi > slots) return -1;
    n += (g.hi - g.lo + size - 1) / size;
  }
  return n;
}
extern "C" int64_t most(int64_t slots, int64_t groups, int64_t size) { return sphops::most_tiles(slots, groups, size); }
extern "C" int64_t places(int64_t tiles, int room) { return sphops::slice_places(tiles, room); }
extern "C" void turns(uint32_t tiles, uint32_t room, uint32_t places, int depth, uint32_t* out) {
  const sphops::Turns t = sphops::turns_of(tiles, room, places, depth);
  out[0] = t.whole;
  out[1] = t.left;
  out[2] = t.slices;
}
"""
ROOM, SIDE = 512, 128  # 16-bit tiles of 128 x 128, of which the card holds 512


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    at = tmp_path_factory.mktemp("turns")
    (at / "turns.hip").write_text(SOURCE)
    subprocess.run([HIPCC, "-x", "hip", "--cuda-host-only", "--offload-arch=gfx950", "-std=c++17", "-O1", "-fPIC", "-shared",
                    "-I", CSRC, str(at / "turns.hip"), "-o", str(at / "turns.so")], check=True, capture_output=True)
    so = ctypes.CDLL(str(at / "turns.so"))
    for name in ("tiles_of", "most", "places"):
        getattr(so, name).restype = ctypes.c_int64
    so.tiles_of.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int64]
    so.most.argtypes = [ctypes.c_int64] * 3
    so.places.argtypes = [ctypes.c_int64, ctypes.c_int]
    so.turns.argtypes = [ctypes.c_uint32] * 3 + [ctypes.c_int, ctypes.c_void_p]
    return so


def _tiles(host, offsets, slots):
    n = host.tiles_of((ctypes.c_int32 * len(offsets))(*offsets), len(offsets) - 1, slots, SIDE)
    assert n >= 0, "rows outside the call's"
    return n


def _turns(host, tiles, places, depth, room=ROOM):
    out = (ctypes.c_uint32 * 3)()
    host.turns(tiles & 0xffffffff, room, places, depth, out)
    return list(out)


def _held(slots, experts, cols, outs):
    """Places of 128 x 128 float32 that the workspace of a bfloat16 layer holds."""
    size = lib.sphops_expert_linear_workspace_bytes(1, slots, experts, cols, outs)
    assert size % (SIDE * SIDE * 4) == 0
    return size // (SIDE * SIDE * 4)


@pytest.mark.parametrize("slots,offsets,depth", [(2000, [0, 2000, 0, 2000], 4096), (500, [0, 500] * 4 + [0], 4096),
                                                 (1200, [0, 1200, 0, 1200, 0], 8192), (1200, [0, 1200] * 10, 4096)])
def test_offsets_that_decrease(host, slots, offsets, depth):
    """More tiles than the workspace was made for: cut by the card's room alone they would leave it."""
    experts = len(offsets) - 1
    held, tiles = _held(slots, experts, depth, SIDE), _tiles(host, offsets, slots)
    assert held == host.places(host.most(slots, experts + 1, SIDE), ROOM) and tiles > host.most(slots, experts + 1, SIDE)
    _, left, slices = _turns(host, tiles, ROOM, depth)
    assert left * slices > held
    _, left, slices = _turns(host, tiles, held, depth)
    assert slices == 1 or left * slices <= held


def test_offsets_of_any_kind(host):
    rng = random.Random(3)
    for _ in range(3000):
        experts, slots, outs = rng.choice([1, 2, 3, 5, 9, 33, 70]), rng.randint(1, 6000), rng.choice([64, 128, 200, 255])
        if slots <= min(1024, 16 * experts):
            continue  # one launch without tiles
        depth = rng.choice([512, 700, 2048, 4096, 9000])
        word = rng.choice([lambda: rng.randint(0, slots), lambda: rng.choice([0, slots]),
                           lambda: rng.randint(-2 ** 31, 2 ** 31 - 1), lambda: rng.randint(-5, slots + 5)])
        offsets = [word() for _ in range(experts + 1)]
        held, nt = _held(slots, experts, depth, outs), -(-outs // SIDE)
        _, left, slices = _turns(host, _tiles(host, offsets, slots) * nt, held, depth)
        assert slices == 1 or left * slices <= held
        # the join's workgroups are the cut tiles
        assert slices == 1 or left <= min(ROOM // 2, held)


def test_offsets_that_do_not_decrease(host):
    """There the workspace is no bound: tiles are cut as the card's room says."""
    rng = random.Random(4)
    for _ in range(3000):
        experts, slots, nt = rng.choice([1, 2, 3, 9, 70]), rng.randint(1, 50000), rng.randint(1, 9)
        offsets = [0, *sorted(rng.randint(0, slots) for _ in range(experts))]
        depth, room = rng.choice([512, 2048, 9000]), rng.choice([256, 512])
        most = host.most(slots, experts + 1, SIDE) * nt
        tiles = _tiles(host, offsets, slots) * nt
        assert tiles <= most
        got = _turns(host, tiles, host.places(most, room), depth, room)
        left = tiles % room
        assert got == [tiles - left, left, max(1, min(room // left, depth // 256, 16)) if left else 1]
