"""Derivatives that the rotation, the cache and the packed attention have not are refused, not dropped (CPU: these checks come
first)."""
import pytest
import torch
from torch.autograd import forward_ad

import omni_attn_torch as oat

Q = torch.zeros(4, 2, 64, dtype=torch.float16)
PAGES = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
I32 = torch.zeros(4, dtype=torch.int32)
TABLE = torch.zeros(4, 64)
W = torch.ones(64, dtype=torch.float16)

CALLS = {
    "rotary": (lambda query=Q, key=Q, table=TABLE, query_norm=W, key_norm=W:
               oat.omni_qk_rotary(query, key, I32, table, query_norm=query_norm, key_norm=key_norm)),
    "append": (lambda query=Q, key=Q, value=Q, key_pages=PAGES, value_pages=PAGES, table=TABLE, query_norm=W, key_norm=W:
               oat.omni_cache_append(key, value, key_pages, value_pages, I32.view(1, 4), I32[:1], I32[:2], table=table, query=query,
                                     query_norm=query_norm, key_norm=key_norm)),
    "packed": lambda query=Q, key=Q, value=Q: oat.omni_attention_packed(query, key, value, I32[:2]),
    "paged": (lambda query=Q, key_pages=PAGES, value_pages=PAGES:
              oat.omni_attention_paged(query, key_pages, value_pages, I32.view(1, 4), I32[:1], I32[:2])),
}
OPERANDS = {
    "rotary": ["query", "key", "table", "query_norm", "key_norm"],
    "append": ["query", "key", "value", "key_pages", "value_pages", "table", "query_norm", "key_norm"],
    "packed": ["query", "key", "value"], "paged": ["query", "key_pages", "value_pages"],
}
PLAIN = {"key_pages": PAGES, "value_pages": PAGES, "table": TABLE, "query_norm": W, "key_norm": W}


@pytest.mark.parametrize("op,name", [(op, name) for op, names in OPERANDS.items() for name in names])
def test_tangents_are_refused(op, name):
    x = PLAIN.get(name, Q)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="forward-mode"):
            CALLS[op](**{name: dual})
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            CALLS[op](**{name: dual})
        with pytest.raises(ValueError, match="GPU tensor"):  # (without tangents the next check speaks)
            CALLS[op]()


@pytest.mark.parametrize("op", ["rotary", "append"])
def test_tables_that_require_a_gradient_are_refused(op):
    learned = TABLE.clone().requires_grad_()
    with pytest.raises(ValueError, match="table must not require a gradient"):
        CALLS[op](table=learned)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU tensor"):  # (nothing is lost: the next check speaks)
        CALLS[op](table=learned)
