"""Host side of the operators for rows that go through different weights: what they refuse, before anything is launched, and the
layout of their descriptors."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000  # stands for a device pointer: every call here is refused, or has no rows, before anything is launched


@pytest.fixture(scope="module")
def bz():
    import blaze_hip
    return blaze_hip


def _fill(desc, **fields):
    d = desc()
    for name, v in fields.items():
        assert hasattr(d, name), name
        setattr(d, name, v)
    return d


def _rc(bz, entry, d):
    rc = getattr(bz.lib(), entry)(C.addressof(d) if d is not None else None, None)
    return rc, bz.lib().bz_last_error().decode()


def _refused(bz, entry, desc, good, changes):
    """each of `changes` makes the good call one that is refused, with a message that names the entry point"""
    rc, text = _rc(bz, entry, None)
    assert rc == bz.EINVAL and entry in text
    for change in changes:
        rc, text = _rc(bz, entry, _fill(desc, **dict(good, **change)))
        assert rc == bz.EINVAL and entry in text, (change, rc, text)


def test_descriptors_match_the_header(tmp_path, bz):
    pairs = {"bz_route_desc": bz.RouteDesc, "bz_group_desc": bz.GroupDesc, "bz_merge_desc": bz.MergeDesc, "bz_merge_grad_desc": bz.MergeGradDesc,
             "bz_grouped_fc_desc": bz.GroupedFcDesc, "bz_fc_adapters_desc": bz.FcAdaptersDesc}
    lines, want = [], []
    for name, desc in pairs.items():
        lines.append('printf("%%zu ", sizeof(%s));' % name)
        want.append(C.sizeof(desc))
        for field, _ in desc._fields_:
            lines.append('printf("%%zu ", offsetof(%s, %s));' % (name, field))
            want.append(getattr(desc, field).offset)
    lines.append('printf("%d %d %d %d %d ", BZ_ROUTE_MAX_N, BZ_ROUTE_MAX_K, BZ_GROUP_MAX_GROUPS, BZ_ADAPTER_MAX_RANK, BZ_ACT_SWIGLU);')
    want += [bz.ROUTE_MAX_N, bz.ROUTE_MAX_K, bz.GROUP_MAX_GROUPS, bz.ADAPTER_MAX_RANK, bz.ACT_SWIGLU]
    src = tmp_path / "s.c"
    src.write_text('#include "blaze_hip.h"\n#include <stdio.h>\nint main(void){%s return 0;}\n' % "".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()] == want


def test_route_topk_refusals(bz):
    good = dict(logits=P, ids=P, weights=P, rows=4, ld=8, n=8, k=2, dtype=bz.F32, score=bz.ROUTE_SOFTMAX, scale=1.0)
    _refused(bz, "bz_route_topk", bz.RouteDesc, good,
             [dict(n=0), dict(n=1025, ld=1025), dict(k=0), dict(k=17, n=32, ld=32), dict(k=9), dict(ld=7), dict(dtype=bz.I32), dict(score=2), dict(rows=-1),
              dict(rows=2**31), dict(logits=None), dict(ids=None), dict(weights=None)])
    assert _rc(bz, "bz_route_topk", _fill(bz.RouteDesc, **dict(good, rows=0, logits=None)))[0] == bz.OK


def test_group_rows_refusals(bz):
    good = dict(ids=P, offsets=P, order=P, position=P, n=64, groups=8)
    moved = dict(good, x=P, xs=P, ld_x=16, ld_xs=16, per=2, dim=16, dtype=bz.F16)
    _refused(bz, "bz_group_rows", bz.GroupDesc, good,
             [dict(n=-1), dict(n=2**31), dict(groups=0), dict(groups=1025), dict(ids=None), dict(order=None), dict(offsets=None),
              dict(n=100000), dict(n=100000, scratch=P, scratch_bytes=16)])
    _refused(bz, "bz_group_rows", bz.GroupDesc, moved,
             [dict(per=0), dict(per=3), dict(dim=0), dict(ld_x=15), dict(ld_xs=15), dict(dtype=bz.I8), dict(xs=None), dict(position=None)])
    assert bz.lib().bz_group_scratch_bytes(64, 8) == 0 and bz.lib().bz_group_scratch_bytes(0, 8) == 0
    for n in (10000, 1 << 20, 2**31 - 1):
        need = bz.lib().bz_group_scratch_bytes(n, 64)
        assert 0 < need <= 64 * 4 * 257


def test_merge_rows_refusals(bz):
    good = dict(xs=P, position=P, weights=P, y=P, rows=4, n=8, ld_xs=16, ld_y=16, k=2, dim=16, dtype=bz.BF16, out_dtype=bz.F32)
    _refused(bz, "bz_merge_rows", bz.MergeDesc, good,
             [dict(k=0), dict(k=17), dict(dim=0), dict(ld_xs=15), dict(ld_y=15), dict(dtype=bz.I64), dict(out_dtype=bz.F16), dict(rows=-1), dict(n=-1),
              dict(rows=2**31), dict(n=2**31), dict(xs=None), dict(position=None), dict(y=None)])
    assert _rc(bz, "bz_merge_rows", _fill(bz.MergeDesc, **dict(good, rows=0)))[0] == bz.OK


def test_merge_rows_grad_refusals(bz):
    good = dict(dy=P, xs=P, position=P, weights=P, dxs=P, dweights=P, rows=4, n=8, ld_dy=16, ld_xs=16, ld_dxs=16, k=2, dim=16, dtype=bz.F16)
    _refused(bz, "bz_merge_rows_grad", bz.MergeGradDesc, good,
             [dict(k=0), dict(k=17), dict(dim=0), dict(ld_dy=15), dict(ld_xs=15), dict(ld_dxs=15), dict(dtype=bz.I32), dict(rows=-1), dict(n=2**31), dict(dy=None),
              dict(xs=None), dict(position=None)])
    assert _rc(bz, "bz_merge_rows_grad", _fill(bz.MergeGradDesc, **dict(good, dxs=None, dweights=None)))[0] == bz.OK


def test_grouped_fc_refusals(bz):
    good = dict(a=P, w=P, bias=P, y=P, offsets=P, a_count=32, lda=16, ldw=16, w_stride=16 * 24, ldy=24, m=32, n=24, k=16, groups=4, rows_per=0,
                in_dtype=bz.F16, out_dtype=bz.F16, act=bz.ACT_NONE)
    _refused(bz, "bz_grouped_fc", bz.GroupedFcDesc, good,
             [dict(m=-1), dict(n=0), dict(k=0), dict(groups=0), dict(groups=1025), dict(lda=15), dict(ldw=15), dict(ldy=23), dict(w_stride=16 * 24 - 1),
              dict(a_count=31), dict(a_count=-1), dict(rows=P, rows_per=0), dict(in_dtype=bz.I8), dict(out_dtype=bz.BF16), dict(act=bz.ACT_SOFTMAX),
              dict(act=7), dict(act=-1), dict(act=bz.ACT_PRELU), dict(act=bz.ACT_PRELU, act_p0=P, act_size=23), dict(act=bz.ACT_DICE, act_p0=P, act_p1=P),
              dict(act=bz.ACT_SWIGLU), dict(a=None), dict(w=None), dict(y=None), dict(offsets=None)])
    assert _rc(bz, "bz_grouped_fc", _fill(bz.GroupedFcDesc, **dict(good, m=0, a=None)))[0] == bz.OK


def test_fc_adapters_refusals(bz):
    good = dict(a=P, w=P, down=P, up=P, scale=P, ids=P, bias=P, y=P, scratch=P, scratch_bytes=32 * 16 * 4, lda=16, ldw=16, ldy=24, ld_down=16, ld_up=8,
                down_stride=8 * 16, up_stride=24 * 8, m=32, n=24, k=16, adapters=4, rank=8, in_dtype=bz.BF16, out_dtype=bz.F32, act=bz.ACT_NONE, alpha=1.0, beta=1.0)
    _refused(bz, "bz_fc_adapters", bz.FcAdaptersDesc, good,
             [dict(m=-1), dict(n=0), dict(k=0), dict(adapters=-1), dict(rank=0), dict(rank=257), dict(lda=15), dict(ldw=15), dict(ldy=23), dict(ld_down=15),
              dict(ld_up=7), dict(down_stride=127), dict(up_stride=191), dict(in_dtype=bz.I32), dict(out_dtype=bz.F16), dict(act=bz.ACT_SOFTMAX),
              dict(act=bz.ACT_SWIGLU), dict(act=bz.ACT_PRELU), dict(act=bz.ACT_DICE), dict(scratch=None), dict(scratch=P + 8), dict(scratch_bytes=32 * 16 * 4 - 1),
              dict(a=None), dict(w=None), dict(down=None), dict(up=None), dict(ids=None), dict(y=None)])
    assert _rc(bz, "bz_fc_adapters", _fill(bz.FcAdaptersDesc, **dict(good, m=0, a=None)))[0] == bz.OK
    size = bz.lib().bz_fc_adapters_scratch_bytes
    assert size(32, 8) == 32 * 16 * 4 and size(1, 256) == 1024 and size(0, 8) == 0 and size(3, 17) == 3 * 32 * 4


@pytest.mark.parametrize("act_size", [1, 23, 25, -1])
def test_dice_of_one_parameter_a_group_is_refused(bz, act_size):
    """Dice has a parameter a column: with fewer, the kernels would read behind them"""
    dice = dict(act=bz.ACT_DICE, act_p0=P, act_p1=P, act_p2=P, n=24, k=16, in_dtype=bz.F16, out_dtype=bz.F16, lda=16, ldw=16, ldy=24)
    for entry, desc, more in (("bz_grouped_fc", bz.GroupedFcDesc, dict(groups=4, w_stride=16 * 24)), ("bz_fc_adapters", bz.FcAdaptersDesc, {})):
        rc, text = _rc(bz, entry, _fill(desc, **dict(dice, **more), act_size=act_size))
        assert rc == bz.EINVAL and entry in text and "Dice" in text
        for whole in (0, 24):
            assert _rc(bz, entry, _fill(desc, **dict(dice, **more), act_size=whole))[0] == bz.OK


def test_the_binding_refuses_dice_of_one_parameter_a_group(bz):
    import torch
    bz._here()  # (what the calls begin with)
    for groups in (1, 3):
        full, one = torch.zeros((groups, 8)), torch.zeros((groups, 1))
        for params in ((one, full, full), (full, one, full), (full, full, one), (one, one, one)):
            with pytest.raises(bz.BlazeHipError, match="act_params.* has %d elements" % groups):
                bz._act_fields("grouped_fc", bz.ACT_DICE, params, 8, groups, -1)
        assert bz._act_fields("grouped_fc", bz.ACT_DICE, (full, full, full), 8, groups, -1)[1] == 8
        assert bz._act_fields("grouped_fc", bz.ACT_PRELU, (one, ), 8, groups, -1)[1] == 1
        with pytest.raises(bz.BlazeHipError, match="act_params"):
            bz._act_fields("grouped_fc", bz.ACT_PRELU, (full, one), 8, groups, -1)


def test_layers_beyond_a_launch_are_refused_before_anything_is_launched(bz):
    """a launch has fewer than 2^32 threads: what would take more is an argument that does not fit, not a launch that fails"""
    layer = dict(a=P, w=P, y=P, in_dtype=bz.F16, out_dtype=bz.F16, k=16, lda=16, ldw=16, act=bz.ACT_NONE)
    sizes = [dict(m=2**31 - 1, n=64, ldy=64), dict(m=2**30, n=64, ldy=64), dict(m=32, n=2**31 - 64, ldy=2**31), dict(m=48, n=2**28, ldy=2**28),
             dict(m=2**20, n=2**17, ldy=2**17), dict(m=2**20, n=2**17, ldy=2**17, in_dtype=bz.F32, out_dtype=bz.F32)]
    for size in sizes:
        # (aligned 2-byte operands within 4 GB have tiles of 256 x 256: 2^37 outputs are 2^21 of them, 2^29 threads, which a launch may have)
        for pitch in (17, ) if size is sizes[4] else (16, 17):
            good = dict(layer, **size)
            good.update(lda=pitch, ldw=pitch)
            rc, text = _rc(bz, "bz_grouped_fc", _fill(bz.GroupedFcDesc, offsets=P, groups=1, a_count=size["m"], **good))
            assert rc == bz.EINVAL and "bz_grouped_fc" in text and "too many" in text, (size, rc, text)
            for adapters in (0, 3):
                rc, text = _rc(bz, "bz_fc_adapters", _fill(bz.FcAdaptersDesc, down=P, up=P, ids=P, scratch=P, scratch_bytes=2**50, ld_down=16, ld_up=8, rank=8,
                                                           adapters=adapters, down_stride=128, up_stride=2**40, alpha=1.0, beta=1.0, **good))
                assert rc == bz.EINVAL and "bz_fc_adapters" in text and "too many" in text, (size, adapters, rc, text)
    gated = dict(layer, m=48, n=2**27, ldy=2**27, act=bz.ACT_SWIGLU)
    rc, text = _rc(bz, "bz_grouped_fc", _fill(bz.GroupedFcDesc, offsets=P, groups=1, a_count=48, **gated))
    assert rc == bz.EINVAL and "too many" in text


def test_tiles_of_offsets_that_run_backwards_stay_in_the_grid(tmp_path):
    """Offsets that go back and forth count a layer's rows up to 512 times, whose tiles times those of its columns pass 32 bits where the layer's
    own do not.  The kernel for many rows counts no further than its launch goes, and with such a count a workgroup has a tile of the grid or none,
    and every tile is one workgroup's."""
    import shutil
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, exe = tmp_path / "tiles.hip", str(tmp_path / "tiles")
    src.write_text(r"""
#include <stdio.h>
#include <vector>
#include "fc_groups.h"
int bz::fail(int code, const char*, ...) { return code; }
using namespace bz::groups;
int main() {
  for (int64_t m : {1, 63, 64, 1000, 1 << 17, 1 << 20})
    for (int groups : {1, 3, 1024})
      for (int tiles_n : {1, 7, 2048, 16384}) {
        const int64_t most = most_tiles(m, groups, 64);
        if ((most * tiles_n + 7) * 256 >= (int64_t)1 << 32) continue;  // (refused on the host)
        if (64 * most >= (int64_t)1 << 31) return 4;  // (what the lanes have counted between them)
        for (int64_t counted : {most, most - 1, most / 2, 512 * (m / 64 + 1)}) {
          const int tiles_m = (int)(counted < most ? counted : most);
          const uint32_t blocks = (uint32_t)((most * tiles_n + 7) / 8 * 8), step = blocks > 1000000 ? 997 : 1;
          std::vector<char> seen(step == 1 && tiles_m > 0 ? (size_t)tiles_m * tiles_n : 0);
          for (uint32_t b = 0; b < blocks; b += step) {
            int tm = -1, tn = -1;
            if (!wide_tile(tiles_m, tiles_n, b, tm, tn)) continue;
            if (tm < 0 || tm >= tiles_m || tn < 0 || tn >= tiles_n) {
              printf("m %lld, %d groups, %d tiles of columns, %lld counted: workgroup %u has tile %d, %d\n", (long long)m, groups, tiles_n, (long long)counted, b, tm, tn);
              return 1;
            }
            if (step == 1 && seen[(size_t)tm * tiles_n + tn]++) return 2;
          }
          for (char c : seen)
            if (c != 1) return 3;
        }
      }
  return 0;
}
""")
    csrc = os.path.join(ROOT, "x-deeplearning_amd", "csrc")
    subprocess.run([hipcc, "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-I" + os.path.join(ROOT, "include"), "-I" + csrc, str(src), "-o", exe],
                   check=True, capture_output=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout)
    # and the kernel counts no further
    assert "reduce<64>(min(tiles, most), [](int a, int b) { return a + b; }), most)" in open(os.path.join(csrc, "fc_groups.h")).read()


def test_a_stream_of_another_device_is_refused(bz):
    """a launch on it would run there, on memory that is here"""
    class Stream:
        device_index, cuda_stream = 1, 0

    def bz_route_topk(desc, stream):
        raise AssertionError("launched")

    with pytest.raises(bz.BlazeHipError, match="bz_route_topk: the stream is of device 1, the current one is 0"):
        bz._call(bz_route_topk, b"", Stream(), 0)
    assert bz.lib().bz_route_topk.__name__ == "bz_route_topk"
