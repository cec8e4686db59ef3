"""The sequence operators' oracle and argument checks on a machine without a GPU."""
import types

import pytest
import torch

import sequence_oracle as R
import sparsl_b200 as S
from sparsl_b200 import _lib

F64 = torch.float64


def _device():
    d = S.Device.__new__(S.Device)
    d._h = None  # no C entry gets past its null check
    return d


def test_oracle_scan_gradients_match_differences():
    g = torch.Generator()
    g.manual_seed(1)
    put = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    lens, ch, ns = [4, 0, 3], 4, 3
    args = [put(7, ch), put(7, ch), -put(ch, ns).abs(), put(7, 2, ns), put(7, 2, ns), put(ch), put(7, ch), put(ch), put(3, ch, ns)]
    for v in args:
        v.requires_grad_()
    f = lambda x, dt, a, b, c, d, z, bias, start: R.scan(x, dt, a, b, c, d, z, bias, True, lens, start)  # noqa: E731
    assert torch.autograd.gradcheck(f, args)


def test_oracle_conv_and_norm_gradients_match_differences():
    g = torch.Generator()
    g.manual_seed(2)
    put = lambda *s: torch.randn(*s, generator=g, dtype=F64).requires_grad_()  # noqa: E731
    assert torch.autograd.gradcheck(lambda x, w, b, s: R.conv(x, w, b, True, [3, 0, 2], s), [put(5, 2), put(2, 4), put(2), put(3, 3, 2)])
    assert torch.autograd.gradcheck(lambda x, w, b: R.norm(x, w, b, 1e-5), [put(3, 5), put(5), put(5)])


def test_magnitudes_bound_the_values():
    g = torch.Generator()
    g.manual_seed(3)
    put = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    lens, ch, ns = [6, 5], 3, 4
    args = dict(x=put(11, ch), dt=put(11, ch), a=-put(ch, ns).abs(), b=put(11, 1, ns), c=put(11, 1, ns), d=put(ch), z=put(11, ch),
                dt_bias=put(ch), start=put(2, ch, ns))
    value = R.scan(softplus=True, lens=lens, **args)
    most = R.scan(softplus=True, lens=lens, magnitude=True, **args)
    for v, m in zip(value, most):
        assert (v.abs() <= m * (1 + 1e-12)).all()


def test_structures_have_the_header_layout(tmp_path):
    import os
    import subprocess

    from conftest import ROOT

    src = tmp_path / "sizes.c"
    names = {"sparsl_conv_args": _lib.ConvArgs, "sparsl_scan_args": _lib.ScanArgs, "sparsl_norm_args": _lib.NormArgs}
    lines = []
    for c, py in names.items():
        lines += [f'printf("%zu\\n", sizeof({c}));'] + [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "sparsl_cuda.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    import ctypes

    want = []
    for py in names.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want


def test_shapes_and_types_are_checked_before_the_library():
    d = _device()
    x, w = torch.zeros(6, 4), torch.zeros(4, 3)
    bad = [
        lambda: d.causal_conv_device(x, torch.zeros(5, 3), x.clone()),
        lambda: d.causal_conv_device(x, w, torch.zeros(6, 5)),
        lambda: d.causal_conv_device(x, w, x.clone(), bias=torch.zeros(3)),
        lambda: d.causal_conv_device(x, w, x.clone(), state=torch.zeros(1, 3, 4)),
        lambda: d.causal_conv_device(x, w, x.clone(), state=torch.zeros(1, 2, 4), final_state=torch.zeros(2, 2, 4)),
        lambda: d.causal_conv_device(x, w, x.clone(), seq_ptr=torch.zeros(3, dtype=torch.int32), slots=torch.zeros(3, dtype=torch.int32)),
        lambda: d.causal_conv_device(x, w, x.clone(), seq_ptr=torch.zeros(3, dtype=torch.int32), n_seq=5),
        lambda: d.layer_norm_device(x, x.clone(), weight=torch.zeros(5)),
        lambda: d.layer_norm_device(x, x.clone(), mean=torch.zeros(5)),
        lambda: d.selective_scan_device(x, x, torch.zeros(5, 2), torch.zeros(6, 2), torch.zeros(6, 2), x.clone()),
        lambda: d.selective_scan_device(x, x, torch.zeros(4, 2), torch.zeros(6, 3), torch.zeros(6, 2), x.clone()),
        lambda: d.selective_scan_device(x, x[:5], torch.zeros(4, 2), torch.zeros(6, 2), torch.zeros(6, 2), x.clone()),
    ]
    for call in bad:
        with pytest.raises(S.OpError) as e:
            call()
        assert e.value.kind == "Length"
    wrong = [
        lambda: d.causal_conv_device(x.double(), w, x.clone()),
        lambda: d.causal_conv_device(x, w, x.half()),
        lambda: d.causal_conv_device(x, w.half(), x.clone()),
        lambda: d.causal_conv_device(x.half(), w.half(), x.half(), bias=torch.zeros(4)),
        lambda: d.causal_conv_device(torch.zeros(4, 6).t(), w, x.clone()),
        lambda: d.causal_conv_device(x, w, x.clone(), seq_ptr=torch.zeros(3, dtype=torch.int64)),
        lambda: d.layer_norm_device(x, x.clone(), mean=torch.zeros(6).half()),
        lambda: d.selective_scan_device(x, x, torch.zeros(4, 2).half(), torch.zeros(6, 2), torch.zeros(6, 2), x.clone()),
        lambda: d.selective_scan_backward_device(x, x, x, torch.zeros(4, 2), torch.zeros(6, 2), torch.zeros(6, 2), None, x.clone(),
                                                 x.clone(), torch.zeros(4, 2), torch.zeros(6, 2), torch.zeros(6, 2), None, z=x),
    ]
    for call in wrong:
        with pytest.raises(TypeError):
            call()


def test_packed_blocks_fill_the_structures():
    """Every field of a packed block lands on its structure's field of that place."""
    import ctypes

    from sparsl_b200 import sequence as Q

    def flat(t, v):
        if isinstance(v, ctypes.Structure):
            return [w for n, f in v._fields_ for w in flat(f, getattr(v, n))]
        return [v or 0]

    for packer, struct in ((Q._CONV, _lib.ConvArgs), (Q._SCAN, _lib.ScanArgs), (Q._NORM, _lib.NormArgs)):
        assert packer.size == ctypes.sizeof(struct)
        count = len(packer.unpack(bytes(packer.size)))
        values = list(range(1, count + 1))
        got = struct.from_buffer_copy(packer.pack(*values))
        assert flat(struct, got) == values


def test_no_device_is_refused():
    d = _device()
    with pytest.raises(S.OpError):
        d.layer_norm_device(torch.zeros(2, 4), torch.zeros(2, 4))


def test_streams_of_torch_map_to_handles():
    from sparsl_b200.sequence import _stream

    assert _stream(None) is None and _stream(77) == 77
    assert _stream(types.SimpleNamespace(cuda_stream=99)) == 99
    assert _stream(types.SimpleNamespace(cuda_stream=0)) == 1  # CUDA's legacy default stream, not the device's own


def test_workspace_sizes():
    D = S.Device
    assert D.causal_conv_backward_workspace(1000, 512, 4) >= 16 * 5 * 512 * 4
    assert D.selective_scan_workspace(64, 2048, 16, 1, 1) == 0  # one chunk
    assert D.selective_scan_workspace(1 << 15, 2048, 16, 1, 1) > 0
    assert D.selective_scan_checkpoints(17, 10, 16) == 3 * 10 * 16 * 4
    assert D.selective_scan_backward_workspace(100, 64, 16, 1, 3) == 0  # 64 channels are no 3 groups: nothing to size
    assert D.layer_norm_backward_workspace(10, 100) == 10 * 2 * 100 * 4


def test_a_handle_is_the_stream_it_comes_from():
    """0, the handle of torch's default stream, is that stream, not the device's own."""
    from sparsl_b200.sequence import _stream

    assert _stream(0) == 1 == _stream(types.SimpleNamespace(cuda_stream=0)) and _stream(1) == 1 and _stream(None) is None


def test_layouts_of_the_scan():
    """Large prompts take one lane a channel and hand states on; whole sequences that fill two fifths of a wave of blocks do not."""
    import ctypes

    def layout(*args):
        out = (ctypes.c_uint64 * 5)()
        assert _lib.load().sparsl_selective_scan_test_layout(*args, out) == 0
        return list(out)

    lanes, chunks, length, carry, first = layout(32768, 2048, 16, 1, 1, 0, 0)
    assert (lanes, carry, first) == (1, 1, 1) and (chunks - 1) * length < 32768 <= chunks * length and length % 32 == 0
    assert layout(16384, 2048, 16, 8, 1, 0, 0) == [2, 8, 2048, 0, 0]
    assert layout(16384, 2048, 16, 8, 1, 0, 1) == [2, 8, 2048, 0, 0]
    assert layout(16384, 2048, 16, 8, 1, 1, 1)[3] == 1  # unequal ones are cut
    for n, back in ((4, 0), (5, 0), (4, 1), (7, 1), (12, 1)):  # whole ones with 4 states a lane, or in waves that stay empty, are slower
        assert layout(n * 2048, 2048, 16, n, 1, 0, back)[3] == 1
    assert layout(7 * 1024, 1024, 64, 7, 1, 0, 0)[3] == 1 and layout(8 * 1024, 1024, 64, 8, 1, 0, 0)[3] == 0
    assert layout(0, 8, 4, 1, 1, 0, 0)[1:2] == [1]
    bad = (ctypes.c_uint64 * 5)()
    for args in ((8, 0, 4, 1, 1, 0, 0), (8, 9, 4, 1, 2, 0, 0), (8, 8, 65, 1, 1, 0, 0), (8, 8, 0, 1, 1, 0, 1)):
        assert _lib.load().sparsl_selective_scan_test_layout(*args, bad) != 0
