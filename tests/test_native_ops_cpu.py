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


def test_tensors_without_memory_are_refused(python):
    """A wrapper's address is 0, or its offset: neither may reach a kernel."""
    said = python("""
freqs, pos = Wrapper(64, dtype=torch.float64), Wrapper(1, 4, dtype=torch.int32)
for offset in (0, 64):
    qkv, half = Wrapper(4, 512, offset=offset), Wrapper(4, 256, offset=offset)
    lse, delta, scratch = (Wrapper(*n, dtype=t, offset=offset) for n, t in (((1, 2, 4), torch.float32), ((1, 2, 4), torch.float32), ((1 << 22,), torch.uint8)))
    print(refused(lambda: ops.rope_apply_axes_(qkv, freqs, pos, 2, 1, 128, (64,))))
    print(refused(lambda: ops.add_rmsnorm_quant(qkv, qkv, Wrapper(512, offset=offset))))
    print(refused(lambda: ops.flash_attn_window_fwd(qkv, 1, 4, 2, 1, 128, 4)))
    print(refused(lambda: ops.flash_attn_window_bwd(qkv, half, half, lse, 1, 4, 2, 1, 128, 4)))
    print(refused(lambda: ops.flash_attn_window_bwd(qkv, half, half, lse, 1, 4, 2, 1, 128, 4, dqkv=Wrapper(4, 512), delta=delta, scratch=scratch)))
""").splitlines()
    assert len(said) == 10 and all("has no memory" in s or "shares memory" in s for s in said), said


@pytest.mark.parametrize("missing", ["x", "g", "q", "scale", "rstd"])
def test_the_norm_launcher_refuses_no_address(missing):
    from cai_b200.ops import KernelError, calls, check
    at = dict(x=1 << 20, ldx=256, residual=0, ldr=0, g=1 << 20, h=0, y=0, q=1 << 20, scale=1 << 20, rstd=1 << 20, rows=4, H=256, eps=1e-6, stream=0)
    at[missing] = 0
    with pytest.raises(KernelError, match="add_rmsnorm_quant: .*null"):
        check(calls().cai_add_rmsnorm_quant(*at.values()), "norm")
    at["rows"] = 0
    assert calls().cai_add_rmsnorm_quant(*at.values()) == 0


@pytest.mark.parametrize("missing", ["qkv", "freqs", "pos"])
def test_the_rotation_launcher_refuses_no_address(missing):
    from cai_b200.ops import KernelError, calls, check
    at = dict(qkv=1 << 20, freqs=1 << 20, pos=1 << 20, ldp=10, T=10, nh=2, nkv=1, hd=128, ld=512, axes=1, n0=64, n1=0, n2=0, n3=0, interleaved=0, inverse=0, stream=0)
    at[missing] = 0
    with pytest.raises(KernelError, match="rope_apply_axes: .*null"):
        check(calls().cai_rope_apply_axes(*at.values()), "rope")
    at["T"] = 0
    assert calls().cai_rope_apply_axes(*at.values()) == 0


@pytest.mark.parametrize("missing", ["qkv", "out", "lse"])
def test_the_window_forward_launcher_refuses_no_address(missing):
    from cai_b200.ops import KernelError, calls, check
    at = dict(qkv=1 << 20, ld=512, out=1 << 20, lse=1 << 20, B=1, S=256, nh=2, nkv=1, hd=128, scale=0.1, window=64, sinks=4, stream=0)
    at[missing] = 0
    with pytest.raises(KernelError, match="flash_attn_window_fwd: .*null"):
        check(calls().cai_flash_attn_window_fwd(*at.values()), "window")
    at["S"] = 0
    assert calls().cai_flash_attn_window_fwd(*at.values()) == 0


@pytest.mark.parametrize("missing", ["qkv", "out", "dout", "lse", "delta", "dqkv"])
def test_the_window_backward_launcher_refuses_no_address(missing):
    from cai_b200.ops import KernelError, calls, check
    at = dict(qkv=1 << 20, ld=512, out=1 << 20, dout=1 << 20, lse=1 << 20, delta=1 << 20, dqkv=1 << 20, ldq=512, scratch=1 << 20, B=1, S=256, nh=2, nkv=1, hd=128, scale=0.1,
              window=64, sinks=4, stream=0)
    at[missing] = 0
    with pytest.raises(KernelError, match="flash_attn_window_bwd: .*null"):
        check(calls().cai_flash_attn_window_bwd(*at.values()), "window")
    at["B"] = 0
    assert calls().cai_flash_attn_window_bwd(*at.values()) == 0
