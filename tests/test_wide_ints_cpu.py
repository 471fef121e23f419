"""Lengths and bounds past 31 bits are refused; the C entries' 32-bit arguments would take them modulo 2^32."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
BIG = 2 ** 32


def fake(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="cuda:0")


def calls():
    """name -> call(n), which hands n to an operator as a length or a bound."""
    from atflash import ops
    i32 = torch.int32
    kv, kv8, exps = fake(8, 2, 2, 2048), fake(8, 2, 2, 2048, dtype=F8), fake(8, 2, 2, dtype=torch.int8)
    q1, q4, rows, kr = fake(2, 4, 128), fake(2, 3, 4, 128), fake(9, 4, 128), fake(9, 2, 128)
    table, cu, lens, one = fake(2, 4, dtype=i32), fake(3, dtype=i32), fake(2, dtype=i32), fake(1, dtype=i32)
    free = fake(8, dtype=i32)
    return {
        "prefill keys": lambda n: ops.prefill(q4, kv, table, 5 + n, 2, None, 0.1, None, 0),
        "prefill offset": lambda n: ops.prefill(q4, kv, table, 5, 2 + n, None, 0.1, None, 0),
        "decode": lambda n: ops.decode_paged(q1, kv, table, lens, 5 + n, None, 0.1, None, 0),
        "plan": lambda n: ops.DecodePlan(kv, table, lens, 5 + n, None, 0.1, None, 0, 4),
        "decode q8": lambda n: ops.decode_paged_q8(q1, kv8, exps, table, lens, 5 + n, None, 0.1, None, 0),
        "expand": lambda n: ops.kv_expand_q8(kv8, exps, table, 1 + n),
        "packed plan rows": lambda n: ops.PackedPlan(cu, lens, 9 + n, 64, 4),
        "packed plan keys": lambda n: ops.PackedPlan(cu, lens, 9, 64 + n, 4),
        "prefill packed": lambda n: ops.prefill_packed(rows, kv, table, cu, lens, 64 + n, None, 0.1, None, 0),
        "flash packed": lambda n: ops.flash_attn_packed(rows, kr, kr, cu, 9 + n, None, 0.1, None, 0),
        "write packed": lambda n: ops.kv_write_packed(kv, None, kr, kr, cu, 9 - 2 * n, lens, table, None, 0),
        "extend rows": lambda n: ops.extend_tables(table, lens, lens, free, one, 5 + n, 8),
        "extend pool": lambda n: ops.extend_tables(table, lens, lens, free, one, 5, 8 + n),
        "release pool": lambda n: ops.release_tables(table, lens, free, one, one, 8 + n),
    }


@pytest.mark.parametrize("n", [BIG, -BIG])
@pytest.mark.parametrize("name", ["prefill keys", "prefill offset", "decode", "plan", "decode q8", "expand", "packed plan rows",
                                  "packed plan keys", "prefill packed", "flash packed", "write packed", "extend rows",
                                  "extend pool", "release pool"])
def test_refused(monkeypatch, name, n):
    from atflash import _lib
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("reached the library"))
    monkeypatch.setattr(_lib, "check", lambda *a: pytest.fail("reached the library"))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 4096)
    with FakeTensorMode():
        if name == "write packed" and n < 0:
            n = -n  # (a large bound is cut to the rows: only one far below zero wraps)
        with pytest.raises(ValueError, match="32 bits"):
            calls()[name](n)
