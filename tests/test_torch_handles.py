"""The shortcuts to torch's current device and stream are optional: without them the public functions are used."""
import importlib.util
import subprocess
import sys

import pytest
import torch

NAMES = ("_cuda_getDevice", "_cuda_getCurrentRawStream")


def test_import_without_the_shortcuts():
    code = "import torch\n" + "".join(f"vars(torch._C).pop('{n}', None)\n" for n in NAMES) + \
        "from cagnet_amd import ops\nassert ops._current_device is torch.cuda.current_device\n"
    subprocess.run([sys.executable, "-c", code], check=True)


@pytest.mark.gpu
def test_both_ways_give_the_same_handles(cuda, monkeypatch):
    from cagnet_amd import ops

    short = ops._current_device, ops._raw_stream
    for n in NAMES:
        monkeypatch.delattr(torch._C, n, raising=False)
    spec = importlib.util.find_spec("cagnet_amd.ops")
    plain = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(plain)
    monkeypatch.undo()  # torch's own public functions call them here
    assert plain._current_device is torch.cuda.current_device
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            assert plain._current_device() == short[0]() == 0
            assert plain._raw_stream(0) == short[1](0) == stream.cuda_stream
            x = torch.ones(3, 5, device=cuda)
            assert torch.equal(plain.rms_norm_fwd(x, None)[0], ops.rms_norm_fwd(x, None)[0])
