"""The timed cases of the operators over several sequences (perf/operators.py): a pass is in order with what its caller
queues before and after it."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture()
def cases():
    import torch

    path = Path(__file__).resolve().parents[1] / "perf" / "operators.py"
    spec = importlib.util.spec_from_file_location("operators_under_test", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    with torch.cuda.stream(torch.cuda.default_stream()):  # (as it was afterwards)
        yield module


@pytest.mark.parametrize("name", ["prompt-ragged", "append-prompts", "decode-batch"])
@pytest.mark.parametrize("own_stream", [False, True])
def test_a_pass_is_in_stream_order(hip, cases, name, own_stream):
    """Outputs cleared ahead of a pass and copied behind it, with no wait in between, on torch's default stream and on
    another: the copy is the pass's result."""
    import torch

    if own_stream:
        torch.cuda.set_stream(torch.cuda.Stream())
    case = next(c for c in cases.listed() if c["name"] == name)
    state = cases.prepare(case, 1)

    def tensors(out):
        return list(out.values()) if isinstance(out, dict) else [out]

    for _ in range(2):
        cases.run(state)
    torch.cuda.synchronize()
    want = [t.clone() for t in tensors(cases.run(state))]
    torch.cuda.synchronize()
    outs = tensors(cases.run(state))
    for _ in range(3):
        big = torch.ones((256 << 20,), device="cuda")
        for _ in range(8):
            big.mul_(1.0)  # (some time for the passes to run ahead of the order)
        for t in outs:
            t.view(torch.uint8).zero_()
        got = [t.clone() for t in tensors(cases.run(state))]
        torch.cuda.synchronize()
        del big
        if name == "append-prompts":  # pages keep what other rows hold: cleared here, the pass's own rows are there
            got, ref = got[:3], want[:3]
        else:
            ref = want
        for x, y in zip(got, ref):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
