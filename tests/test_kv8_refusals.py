"""The 8-bit cache's entry points refuse bad arguments before any launch (no
device needed)."""

import pytest

import feattn

A = 1 << 20  # an aligned address that is never followed


class T:
    """A tensor by its address alone."""

    def __init__(self, at=A):
        self.at = at

    def data_ptr(self):
        return self.at


def call(name, **over):
    t = dict(q=T(), k=T(), v=T(), qkv=T(), k_cache=T(), v_cache=T(), scales=T(), pos=T(), slots=T(), cache=T(),
             q_weight=T(), k_weight=T(), q_out=T(), k_out=T(), v_out=T(), row_stride=48 * 128, eps=1e-6, rows=3,
             hq=32, hkv=8, dim=128, bf16=True, max_positions=64, cache_slots=64)
    if name == "rope_append_kv8":
        t["q"] = T(2 * A)
    t.update(over)
    args = {
        "store_kv8": ("k", "v", "k_cache", "v_cache", "scales", "slots", "rows", "hkv", "dim", "bf16", "cache_slots"),
        "rope_append_kv8": ("q", "k", "v", "k_cache", "v_cache", "scales", "pos", "slots", "cache", "rows", "hq",
                            "hkv", "dim", "bf16", "max_positions", "cache_slots"),
        "norm_rope_append_kv8": ("qkv", "row_stride", "q_weight", "k_weight", "eps", "q_out", "k_cache", "v_cache",
                                 "scales", "pos", "slots", "cache", "rows", "hq", "hkv", "bf16", "max_positions",
                                 "cache_slots", "dim"),
        "load_kv8": ("k_cache", "v_cache", "scales", "slots", "k_out", "v_out", "rows", "hkv", "dim", "bf16",
                     "cache_slots"),
    }[name]
    return getattr(feattn, name)(*[t[a] for a in args], stream=0)


NAMES = ("store_kv8", "rope_append_kv8", "norm_rope_append_kv8", "load_kv8")
TENSORS = {
    "store_kv8": ("k", "v", "k_cache", "v_cache", "scales", "slots"),
    "rope_append_kv8": ("q", "k", "v", "k_cache", "v_cache", "scales", "pos", "slots", "cache"),
    "norm_rope_append_kv8": ("qkv", "q_weight", "k_weight", "q_out", "k_cache", "v_cache", "scales", "pos", "slots",
                             "cache"),
    "load_kv8": ("k_cache", "v_cache", "scales", "slots", "k_out", "v_out"),
}


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("over,says", [({"rows": -1}, "negative"), ({"hkv": -1}, "negative"),
                                       ({"cache_slots": -16}, "negative"), ({"dim": 64}, "128"),
                                       ({"cache_slots": 72}, "multiple of 16")])
def test_sizes(name, over, says):
    with pytest.raises(RuntimeError, match=says):
        call(name, **over)


@pytest.mark.parametrize("name,tensor", [(n, t) for n in NAMES for t in TENSORS[n]])
def test_null_and_misaligned(name, tensor):
    with pytest.raises(RuntimeError, match="null"):
        call(name, **{tensor: T(0)})
    if tensor not in ("pos", "slots"):
        with pytest.raises(RuntimeError, match="aligned"):
            call(name, **{tensor: T(A + 4)})


def test_queries_apart():
    with pytest.raises(RuntimeError, match="negative"):
        call("rope_append_kv8", hq=-1)
    with pytest.raises(RuntimeError, match="negative"):
        call("norm_rope_append_kv8", hq=-1)
    with pytest.raises(RuntimeError, match="alias"):
        call("rope_append_kv8", q=T())
    with pytest.raises(RuntimeError, match="row_stride"):
        call("norm_rope_append_kv8", row_stride=47 * 128)
    with pytest.raises(RuntimeError, match="row_stride"):
        call("norm_rope_append_kv8", row_stride=48 * 128 + 4)


@pytest.mark.parametrize("name", NAMES)
def test_nothing_to_do(name):
    call(name, rows=0)
    call(name, hkv=0, **({"hq": 0} if "append" in name else {}))


def test_attention_needs_a_plan():
    lib = feattn.lib()
    assert lib.fe_attn_run_kv8(None, A, A, A, A, A, None, 1, None) == feattn.FE_EINVAL
    assert b"plan" in lib.fe_attn_last_error()
