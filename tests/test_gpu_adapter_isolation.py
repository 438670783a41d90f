"""One request's adapter does not reach another's rows, whatever stands in it."""
import pytest
import torch

from mantle_b200 import head as H
from test_gpu_head import BF16, E4M3, head_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 40, 128, 300])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("beside", [False, True])
def test_an_adapter_that_is_not_finite_spoils_its_own_rows_only(rows, dtype, beside):
    s = head_inputs(rows, 700, 128, dtype, 4, 24, beside=beside)
    s["ids"].copy_(torch.arange(rows, dtype=torch.int32) % 5 - 1)

    def run(a, b, replaced=False):
        table = H.Adapters(s["a"].clone() if replaced else a, s["b"] if replaced else b, s["gain"])
        if replaced:
            table.replace(2, a[2], b[2], float(s["gain"][2]))
        got = H.HeadPlan(s["hidden"], s.get("weight"), hidden_scales=s.get("hidden_scales"), weight_scales=s.get("weight_scales"),
                         adapters=table, adapter_ids=s["ids"], base=s.get("base")).launch()
        torch.cuda.synchronize()
        return got

    clean = run(s["a"], s["b"])
    keep = s["ids"] != 2
    for value in (float("inf"), float("-inf"), float("nan")):
        for where in ("a", "b"):
            bad = {"a": s["a"].clone(), "b": s["b"].clone()}
            bad[where][2, 3::7] = value
            for replaced in (False, True):
                got = run(bad["a"], bad["b"], replaced)
                assert torch.equal(got[keep], clean[keep]), (value, where, replaced)
                if bool((~keep).any()):
                    assert not torch.equal(got[~keep], clean[~keep])


@pytest.mark.parametrize("gain", ["much", None, [1.0, 2.0], torch.ones(2)])
def test_a_refused_replacement_leaves_the_table_as_it_was(gain):
    s = head_inputs(10, 300, 128, BF16, 3, 8)
    t = head_inputs(10, 300, 128, BF16, 3, 8, seed=40)
    table = H.Adapters(s["a"], s["b"], s["gain"])
    kept = [x.clone() for x in (table.a, table.gain, table.packed)]
    with pytest.raises((TypeError, ValueError)):
        table.replace(1, t["a"][0], t["b"][0], gain)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(kept, (table.a, table.gain, table.packed)))
