"""The paged key-value cache's operators have no gradient: every input that asks for one is refused,
unless gradients are off."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def tensors(cache):
    z = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    scaled = cache == torch.float8_e4m3fn
    rows = torch.float16 if scaled else cache
    a = {"q": z(1, 4, 64, dtype=rows), "k": z(1, 2, 64, dtype=rows), "v": z(1, 2, 64, dtype=rows),
         "k_pages": z(3, 2, 16, 64, dtype=cache), "v_pages": z(3, 2, 16, 64, dtype=cache), "weights": z(3, 2, 16),
         "cos_sin": z(4, 64)}
    if scaled:
        a["k_scale"], a["v_scale"] = z(3, 2, 16), z(3, 2, 16)
    ints = {"index_pages": z(3, 2, 16, dtype=torch.int32), "table": z(1, 2, dtype=torch.int32),
            "lengths": torch.full((1,), 20, dtype=torch.int32, device="cuda"), "slots": torch.arange(1).cuda(),
            "positions": z(1, dtype=torch.int32)}
    return a, ints


def calls(a, i):
    from pynve.torch import nve_kv

    scales = {n: a[n] for n in ("k_scale", "v_scale") if n in a}
    return {
        "append": lambda: nve_kv.kv_append(a["k"], a["v"], a["k_pages"], a["v_pages"], i["slots"], q=a["q"],
                                           positions=i["positions"], cos_sin=a["cos_sin"], weights=a["weights"],
                                           index_pages=i["index_pages"], **scales),
        "attend": lambda: nve_kv.kv_attend(a["q"], a["k_pages"], a["v_pages"], i["table"], i["lengths"],
                                           weights=a["weights"], **scales),
        "attend_lse": lambda: nve_kv.kv_attend(a["q"], a["k_pages"], a["v_pages"], i["table"], i["lengths"],
                                               weights=a["weights"], return_lse=True, **scales),
        "evict": lambda: nve_kv.kv_evict(a["k_pages"], a["v_pages"], a["weights"], i["index_pages"], i["table"],
                                         i["lengths"], 8, **scales),
    }


READ = {"append": ["q", "k", "v", "cos_sin"], "attend": ["q"], "attend_lse": ["q"], "evict": []}


@pytest.mark.parametrize("op", list(READ))
@pytest.mark.parametrize("cache", [torch.float32, torch.float16, torch.float8_e4m3fn])
def test_inputs_that_ask_for_a_gradient(op, cache):
    a, ints = tensors(cache)
    calls(a, ints)[op]()
    names = READ[op] + ["k_pages", "v_pages", "weights"] + [n for n in ("k_scale", "v_scale") if n in a]
    for name in names:
        asks = {**a, name: a[name].clone().requires_grad_()}
        with pytest.raises(RuntimeError, match=f"{name} asks for a gradient"):
            calls(asks, ints)[op]()
        with torch.no_grad():
            calls(asks, ints)[op]()
