"""Child process of test_batch_edges_gpu.py: prints which kernels the shared-prefix attention launches for its steps, as JSON."""

import json
import pathlib
import sys

HERE = pathlib.Path(__file__).resolve().parent
sys.path[:0] = [str(HERE), str(HERE.parent), str(HERE.parent / "iree-adreno-genai-tuner_b200")]

import torch  # noqa: E402
from torch.profiler import ProfilerActivity, profile  # noqa: E402

import q4b  # noqa: E402
from test_batch_edges_gpu import _attend_case, _dev, _odd, _steps  # noqa: E402


def kernels(call):
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    return sorted({e.key for e in prof.key_averages() if "prefix_" in e.key})


def main():
    out = {}
    for name, (args, kw) in _steps().items():
        b, q, kp, vp = _attend_case(*args, 5)
        d = _dev(b)
        call = lambda x: q4b.prefix_attention(x, kp, vp, d["prefix_pages"], b["prefix_len"], d["page_table"],  # noqa: E731
                                              d["seq_lens"], d["q_start"], **kw)
        out[name] = kernels(lambda: call(q))
        out[name + " odd"] = kernels(lambda: call(_odd(q)))
    print(json.dumps(out))


if __name__ == "__main__":
    main()
