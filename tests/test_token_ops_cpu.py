"""Token-block operators without a GPU: fake shapes of the registered ops, refusals before any launch, and
the host side of the C entry points (argument checks, workspace sizes)."""
import random
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mragan_hip.torch_ops  # noqa: F401
from mragan_hip import MraganError, ops
from mragan_hip._lib import call, query


def test_fake_shapes():
    m = torch.ops.mragan
    with FakeTensorMode():
        x = torch.empty(2, 4, 4, 4, 96, dtype=torch.bfloat16)
        y, mean, rstd = m.layer_norm(x, torch.empty(96), None, 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == rstd.shape == (2, 4, 4, 4) and mean.dtype == torch.float32
        w = [torch.empty(s, dtype=torch.bfloat16) for s in ((200, 96), (200, 96), (48, 200))]
        y, kept = m.gated_ffn(x, *w, None, None, None, "silu", True)
        assert y.shape == (2, 4, 4, 4, 48) and kept.shape == (4, 128, 200) and kept.dtype == torch.bfloat16
        assert m.gated_ffn(x, *w, None, None, None, "silu", False)[1].numel() == 0
        s = torch.empty(3, 300, 96)
        y, last, carry = m.linear_recurrence(s, s, None, None, False)
        assert y.shape == s.shape and last.shape == (3, 96) and carry.shape == (3, 3, 96)


def test_cpu_tensors_refused():
    x = torch.zeros(2, 3, 8)
    w = torch.zeros(16, 8)
    for fn in (lambda: ops.layer_norm_fwd(x), lambda: ops.gated_ffn_fwd(x, w, w, w.t()), lambda: ops.linear_recurrence_fwd(x, x),
               lambda: ops.layer_norm_bwd(x, x[..., 0], x[..., 0], x), lambda: ops.linear_recurrence_bwd(x, x, x, x)):
        with pytest.raises(ValueError, match="device tensor"):
            fn()
    with pytest.raises(Exception):
        torch.ops.mragan.layer_norm(x, None, None, 1e-5)


P = 1 << 20      # an aligned address that is never dereferenced: each call below is refused on the host


@pytest.mark.parametrize("match,name,args", [
    ("null pointer", "mragan_layer_norm_fwd", (None, 4, 8, 0, None, None, 0, 1e-5, P, P, P, None)),
    ("bad shape", "mragan_layer_norm_fwd", (P, 4, 0, 0, None, None, 0, 1e-5, P, P, P, None)),
    ("bad shape", "mragan_layer_norm_fwd", (P, -1, 8, 0, None, None, 0, 1e-5, P, P, P, None)),
    ("bad types", "mragan_layer_norm_fwd", (P, 4, 8, 3, None, None, 0, 1e-5, P, P, P, None)),
    ("bad types", "mragan_layer_norm_fwd", (P, 4, 8, 0, None, None, 1, 1e-5, P, P, P, None)),
    ("eps", "mragan_layer_norm_fwd", (P, 4, 8, 0, None, None, 0, -1.0, P, P, P, None)),
    ("too many rows", "mragan_layer_norm_fwd", (P, 1 << 31, 8, 0, None, None, 0, 1e-5, P, P, P, None)),
    ("workspace", "mragan_layer_norm_bwd", (P, P, P, P, 4, 8, 0, P, 0, P, P, P, None, 0, None)),
    ("null pointer", "mragan_layer_norm_bwd", (P, None, P, P, 4, 8, 0, P, 0, P, P, P, P, 1 << 20, None)),
    ("null pointer", "mragan_gated_ffn_fwd", (P, 4, 8, 8, 8, 0, P, None, P, None, None, None, 5, P, None, P, 1 << 40, None)),
    ("bad shape", "mragan_gated_ffn_fwd", (P, 4, 8, 0, 8, 0, P, P, P, None, None, None, 5, P, None, P, 1 << 40, None)),
    ("activation", "mragan_gated_ffn_fwd", (P, 4, 8, 8, 8, 0, P, P, P, None, None, None, 7, P, None, P, 1 << 40, None)),
    ("dtype", "mragan_gated_ffn_fwd", (P, 4, 8, 8, 8, -1, P, P, P, None, None, None, 5, P, None, P, 1 << 40, None)),
    ("aligned", "mragan_gated_ffn_fwd", (P + 8, 4, 8, 8, 8, 0, P, P, P, None, None, None, 5, P, None, P, 1 << 40, None)),
    ("workspace", "mragan_gated_ffn_fwd", (P, 4, 8, 8, 8, 0, P, P, P, None, None, None, 5, P, None, P, 64, None)),
    ("side above", "mragan_gated_ffn_fwd", (P, (1 << 30) + 1, 8, 8, 8, 0, P, P, P, None, None, None, 5, P, None, P, 1 << 60, None)),
    ("side above", "mragan_gated_ffn_fwd", (P, 4, 1 << 22, 8, 8, 0, P, P, P, None, None, None, 5, P, None, P, 1 << 40, None)),
    ("no rows", "mragan_gated_ffn_bwd", (P, 0, 8, 8, 8, 0, P, P, P, None, None, 5, P, None) + (P,) * 7 + (P, 1 << 40, None)),
    ("workspace", "mragan_gated_ffn_bwd", (P, 4, 8, 8, 8, 0, P, P, P, None, None, 5, P, None) + (P,) * 7 + (P, 64, None)),
    ("bad shape", "mragan_linear_recurrence_fwd", (P, 8, 8, P, 8, 8, None, 0, 0, None, 1, 0, 8, 0, 0, P, P, P, None, 0, None)),
    ("reverse", "mragan_linear_recurrence_fwd", (P, 8, 8, P, 8, 8, None, 0, 0, None, 1, 4, 8, 0, 2, P, P, P, None, 0, None)),
    ("time strides", "mragan_linear_recurrence_fwd", (P, 8, 1 << 22, P, 8, 8, None, 0, 0, None, 1, 4, 8, 0, 0, P, P, P, None, 0, None)),
    ("time strides", "mragan_linear_recurrence_fwd", (P, 8, -8, P, 8, 8, None, 0, 0, None, 1, 4, 8, 0, 0, P, P, P, None, 0, None)),
    ("null pointer", "mragan_linear_recurrence_fwd", (P, 8, 8, None, 8, 8, None, 0, 0, None, 1, 4, 8, 0, 0, P, P, P, None, 0, None)),
    ("null pointer", "mragan_linear_recurrence_fwd", (P, 8, 8, P, 8, 8, None, 0, 0, None, 1, 4, 8, 0, 0, P, None, P, None, 0, None)),
    ("too many", "mragan_linear_recurrence_fwd", (P, 8, 8, P, 8, 8, None, 0, 0, None, 1 << 40, 4, 8, 0, 0, P, P, P, None, 0, None)),
    ("too many", "mragan_linear_recurrence_fwd", (P, 8, 8, P, 8, 8, None, 0, 0, None, 1 << 23, 17, 64, 0, 0, P, P, P, None, 0, None)),
    ("too many", "mragan_linear_recurrence_fwd", (P, 8, 8, P, 8, 8, None, 0, 0, None, 1 << 32, 1, 4, 0, 0, P, P, P, None, 0, None)),
    ("too many rows or channels", "mragan_layer_norm_fwd", (P, 1, (1 << 30) + 1, 0, None, None, 0, 1e-5, P, P, P, None)),
    ("too many rows or channels", "mragan_layer_norm_bwd", (P, P, P, P, 1 << 31, 8, 0, None, 0, P, None, None, None, 0, None)),
    ("without a gate", "mragan_linear_recurrence_bwd", (P, 8, 8, P, 8, 8, None, 0, 0, P, P, 8, 8, None, 1, 4, 8, 0, 0, P, P, P, P, None, 0, None)),
])
def test_entry_points_refuse(match, name, args):
    with pytest.raises(MraganError, match=match):
        call(name, *args)


def test_nothing_to_do_is_no_error():
    call("mragan_layer_norm_fwd", None, 0, 8, 0, None, None, 0, 1e-5, None, None, None, None)
    call("mragan_gated_ffn_fwd", None, 0, 8, 8, 8, 0, None, None, None, None, None, None, 5, None, None, None, 0, None)
    call("mragan_linear_recurrence_fwd", P, 8, 8, P, 8, 8, None, 0, 0, None, 0, 4, 8, 0, 0, None, None, None, None, 0, None)
    call("mragan_layer_norm_bwd", P, P, P, P, 4, 8, 0, None, 0, None, None, None, None, 0, None)


def test_workspace_sizes():
    assert query("mragan_layer_norm_bwd_workspace", 0, 8, 0) == 0
    assert query("mragan_layer_norm_bwd_workspace", 100, 64, 0) >= 2 * 64 * 4
    assert query("mragan_gated_ffn_workspace", 0, 8, 8, 8, 0, 0, 0) == 0
    fwd, bwd, again = (query("mragan_gated_ffn_workspace", 512, 128, 256, 128, 1, b, r) for b, r in ((0, 0), (1, 0), (1, 1)))
    assert 512 * 256 * 2 <= fwd < bwd < again
    try:                                    # fp32 tensors: one 16-bit plane an operand, or three
        sizes = []
        for mode in ("bf16", "bf16x3", "f32"):
            ops.set_conv_precision(mode)
            sizes.append(query("mragan_gated_ffn_workspace", 512, 128, 256, 128, 0, 1, 0))
        assert sizes[0] < sizes[1] < sizes[2]
    finally:
        ops.set_conv_precision("f32")
    assert query("mragan_linear_recurrence_workspace", 1, 16, 64, 0) == 0
    assert query("mragan_linear_recurrence_workspace", 1, 65536, 64, 0) > 0
    assert [query("mragan_linear_recurrence_carries", t, 8) for t in (0, 1, 128, 129)] == [0, 1, 1, 2]


def test_gated_ffn_bwd_workspace_covers_every_subset():
    """The queried size is enough for any choice of gradients: what each choice takes is read from the refusal of a
    call without a workspace, which launches nothing."""
    rng = random.Random(5)
    size = lambda lo, hi, step: max(step, int(lo * (hi / lo) ** rng.random()) // step * step)
    shapes = [(1024, 512, 1024, 512), (512, 512, 1024, 512), (4096, 1024, 1024, 1024), (4096, 1024, 1024, 64), (1, 1, 1, 1),
              (16384, 2048, 8192, 2048), (257, 515, 333, 130), (3, 5, 7, 11)]
    shapes += [(size(1, 16384, 1), *(size(8, hi, rng.choice((1, 8, 64))) for hi in (2048, 8192, 2048))) for _ in range(72)]
    short = []
    try:
        for dtype, mode in ((1, "f32"), (2, "f32"), (0, "f32"), (0, "bf16x3"), (0, "bf16"), (0, "fp16")):
            ops.set_conv_precision(mode)
            for M, C, F, O in shapes:
                for kept in (None, 5 * P):
                    have = query("mragan_gated_ffn_workspace", M, C, F, O, dtype, 1, int(kept is None))
                    for need in range(1, 128):
                        grads = [P if need >> k & 1 else None for k in range(7)]
                        with pytest.raises(MraganError, match="workspace") as e:
                            call("mragan_gated_ffn_bwd", P, M, C, F, O, dtype, P, 2 * P, 3 * P, None, None, 5, 4 * P, kept, *grads,
                                 None, 0, None)
                        takes = int(re.search(r"workspace 0 < (\d+) bytes", str(e.value)).group(1))
                        if takes > have:
                            short.append((dtype, mode, M, C, F, O, kept is None, need, takes - have))
    finally:
        ops.set_conv_precision("f32")
    assert not short, (len(short), short[:5])


def test_single_position_has_no_time_stride():
    """A position of a time-major tensor: torch calls it contiguous whatever the stride of its only step."""
    big = torch.empty(3, 1024, 4096, dtype=torch.bfloat16, device="meta")
    x = big[1:2].transpose(0, 1)
    assert x.stride() == (4096, 1024 * 4096, 1) and x.is_contiguous()
    t, sb, st = ops._sequence(x, "x", x)
    assert t is x and sb == 4096 and 0 <= st < 1 << 22
    for st in (1 << 40, -8):                                  # past the strides' check: the next one refuses
        with pytest.raises(MraganError, match="null pointer"):
            call("mragan_linear_recurrence_fwd", P, 8, st, P, 8, st, P, 8, st, None, 1, 1, 8, 0, 0, None, None, None, None, 0, None)
        with pytest.raises(MraganError, match="without a gate"):
            call("mragan_linear_recurrence_bwd", P, 8, st, P, 8, st, None, 0, st, P, P, 8, st, None, 1, 1, 8, 0, 0, P, P, P, P, None, 0,
                 None)


def test_recurrence_rows_up_to_2_25():
    """A scan along the depth of a volume has H·W·C channels: 2^22 of them are a 256 x 256 plane of 64.  The first two
    calls pass the strides' check and are refused by the next one."""
    for C in (1 << 22, (1 << 25) - 1):
        with pytest.raises(MraganError, match="null pointer"):
            call("mragan_linear_recurrence_fwd", P, 0, C, P, 0, C, P, 0, C, None, 1, 40, C, 0, 0, None, None, None, P, 1 << 50, None)
        with pytest.raises(MraganError, match="without a gate"):
            call("mragan_linear_recurrence_bwd", P, 0, C, P, 0, C, None, 0, 0, P, P, 0, C, None, 1, 40, C, 0, 0, P, P, P, P, P, 1 << 50,
                 None)
        with pytest.raises(MraganError, match="time strides"):
            call("mragan_linear_recurrence_fwd", P, 0, C, P, 0, 3 * C, P, 0, C, None, 1, 40, C, 0, 0, P, P, P, P, 1 << 50, None)
    for T in (1, 40):
        with pytest.raises(MraganError, match="time strides"):
            call("mragan_linear_recurrence_fwd", P, 0, 1 << 25, P, 0, 1 << 25, P, 0, 1 << 25, None, 1, T, 1 << 25, 0, 0, P, P, P, P,
                 1 << 50, None)
    rows = torch.empty(2, 40, 1 << 22, dtype=torch.bfloat16, device="meta")
    t, sb, st = ops._sequence(rows, "x", rows)
    assert t is rows and (sb, st) == (40 << 22, 1 << 22)
    part = torch.empty(2, 40, 3 << 22, dtype=torch.bfloat16, device="meta")[..., :1 << 22]
    assert ops._sequence(part, "x", rows)[1:] == (40 << 22, 1 << 22)
