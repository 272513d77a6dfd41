"""The 8-bit operators' bindings, without a GPU: extents that the library's 32-bit arguments do not hold are refused, not cut to their low bits."""
import json
import os
import subprocess
import types

import pytest

from webdnn_amd import hostops as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HUGE = 2 ** 32 + 5


def tensor(*dims, data_type="float32"):
    length = 1
    for d in dims:
        length *= d
    return types.SimpleNamespace(dims=list(dims), ndim=len(dims), data_type=data_type, length=length, handle=1)


E4M3 = "float8e4m3fn"
BLOCKS = -(-HUGE // 128)


@pytest.mark.parametrize("call", [
    lambda: H.quantize_fp8(None, tensor(1, HUGE), out=(tensor(1, HUGE, data_type=E4M3), tensor(1, BLOCKS))),
    lambda: H.rms_normalization(None, tensor(1, HUGE), out=(None, tensor(1, HUGE))),
    lambda: H.rms_normalization_fp8(None, tensor(1, HUGE), out=(None, tensor(1, HUGE, data_type=E4M3), tensor(1, BLOCKS))),
    lambda: H.matmul_fp8(None, tensor(1, HUGE, data_type=E4M3), tensor(1, BLOCKS), tensor(3, HUGE, data_type=E4M3), tensor(1, BLOCKS), out=tensor(1, 3)),
    lambda: H.matmul_fp8(None, tensor(1, 3, data_type=E4M3), tensor(1, 1), tensor(HUGE, 3, data_type=E4M3), tensor(BLOCKS, 1), out=tensor(1, HUGE)),
    lambda: H.cache_append(None, H.KvCache(None, tensor(HUGE, 1, 64, 32, data_type=E4M3), tensor(HUGE, 1), tensor(HUGE, 1, 32, 64, data_type=E4M3), tensor(HUGE, 1)),
                           tensor(1, 32), tensor(1, 32), tensor(1, 1, data_type="int32"), tensor(1, data_type="int32"), tensor(2, data_type="int32")),
    lambda: H.cache_attention(None, H.KvCache(None, tensor(2, 1, 64, 32, data_type=E4M3), tensor(2, 1), tensor(2, 1, 32, 64, data_type=E4M3), tensor(2, 1)),
                              tensor(HUGE, 32), 1, 1.0, tensor(1, 1, data_type="int32"), tensor(1, data_type="int32"), tensor(2, data_type="int32"),
                              out=tensor(HUGE, 32)),
])
def test_python_refuses_what_32_bits_do_not_hold(call, monkeypatch):
    monkeypatch.setattr(H, "call", lambda name, *args: pytest.fail("%s%r was called" % (name, args)))
    with pytest.raises(H.OperatorError) as err:
        call()
    assert "32 bits" in str(err.value)


def test_javascript_refuses_what_32_bits_do_not_hold():
    code = """
const n = require("./webdnn_amd/lib/webdnn_hip.node"), huge = 2 ** 32 + 5, told = [];
const one = Array(19).fill(1);
const calls = [["rmsnorm", 10, [8]], ["quantizeFp8", 6, [4, 5]], ["gemmFp8", 11, [7, 8, 9]], ["cacheAppend", 19, [13, 14, 15, 16, 17, 18]],
               ["cacheAttention", 19, [11, 12, 13, 14, 15, 16, 17]]];
for (const [name, count, places] of calls)
  for (const at of places)
    for (const value of [huge, -huge, 2 ** 31]) {
      const args = one.slice(0, count);
      args[at] = value;
      try { n[name](...args); told.push("none"); } catch (e) { told.push(e.message); }
    }
console.log(JSON.stringify(told));
"""
    out = subprocess.run(["node", "-e", code], cwd=ROOT, stdout=subprocess.PIPE, text=True, check=True, timeout=60).stdout
    told = json.loads(out.strip().splitlines()[-1])
    assert len(told) == 57 and all("32 bits" in message for message in told), told
