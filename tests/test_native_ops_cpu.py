"""The native operators on tensors that have no memory, in a process of its own without a GPU: a small library in front of torch's answers that device 0 is the current one,
so that the checks behind that one are reached."""
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

DEVICES = """
#include <c10/cuda/CUDAStream.h>
namespace c10::cuda {
DeviceIndex current_device() { return 0; }
CUDAStream getCurrentCUDAStream(DeviceIndex) { return CUDAStream(CUDAStream::UNCHECKED, c10::Stream(c10::Stream::DEFAULT, c10::Device(c10::kCUDA, 0))); }
}
"""

# tensors that say they are on the GPU and have no address
TENSORS = """
import torch
from cai_b200 import ops

class Wrapper(torch.Tensor):
    @staticmethod
    def __new__(cls, *size, dtype=torch.bfloat16, offset=0):
        return torch.Tensor._make_wrapper_subclass(cls, size, strides=torch.empty(size, device="meta").stride(), storage_offset=offset, dtype=dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))

def refused(call):
    try:
        call()
    except RuntimeError as e:          # KernelError is one
        assert not isinstance(e, NotImplementedError) and "launch failed" not in str(e), e
        return str(e)
    raise AssertionError("taken")
"""


@pytest.fixture(scope="module")
def python(tmp_path_factory):
    """Runs a program behind the library; its output."""
    import torch
    from cai_b200 import _build
    where = tmp_path_factory.mktemp("devices")
    (where / "devices.cc").write_text(DEVICES)
    include = Path(torch.__file__).parent / "include"
    cuda = Path(_build.NVCC).resolve().parent.parent / "include"
    if not Path(sysconfig.get_paths()["include"], "Python.h").exists():
        pytest.skip("built without the extension")
    subprocess.run([_build.CXX, "-std=c++17", "-shared", "-fPIC", "-isystem", include, "-isystem", cuda, where / "devices.cc", "-o", where / "devices.so"], check=True)

    def run(program):
        env = dict(os.environ, LD_PRELOAD=str(where / "devices.so"), PYTHONPATH=str(ROOT), CUDA_VISIBLE_DEVICES="")
        done = subprocess.run([sys.executable, "-c", TENSORS + program], env=env, capture_output=True, text=True, timeout=300)
        assert done.returncode == 0, done.stderr[-2000:]
        return done.stdout
    return run


def test_a_tensor_without_storage_is_an_error(python):
    """Under torch.vmap a tensor has no address, and asking for it throws: that becomes a Python exception, and the process goes on, other threads too."""
    assert python("""
import threading
freqs, pos = Wrapper(64, dtype=torch.float64), Wrapper(1, 4, dtype=torch.int32)

def rows(qkv):
    print(refused(lambda: ops.rope_apply_axes_(qkv, freqs, pos, 2, 1, 128, (64,))))
    return qkv
torch.vmap(rows)(Wrapper(2, 4, 512))
t = threading.Thread(target=lambda: print("thread"))
t.start()
t.join()
""").splitlines()[-1] == "thread"
