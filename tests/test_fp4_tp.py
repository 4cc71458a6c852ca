"""CPU, world_size 2 over gloo: dit.TPW4A4MLP on several ranks, its operators replaced
by the 64-bit restatement (oracle/fp4_oracle.py) in each rank's own process.

fc1 is column-parallel: a weight row keeps its scales when the rows are sharded, so the
ranks' hidden columns are the unsharded ones.  fc2 quantises the local K slice of weight
and activations, rank 0 adds the bias, and the bf16 partials are summed over the group.
"""
from __future__ import annotations

import pickle
import traceback
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import fp4_oracle as f4
from test_tp_gloo import _init, _run

TOKENS, D, FFN, SEED = 12, 64, 192, 5
DTYPE = {"nvfp4": torch.float8_e4m3fn, "mxfp4": torch.float8_e8m0fnu}


def _quant(x: torch.Tensor, fmt: str):
    codes, tiles, rows = f4.quantise(x, fmt)
    return (torch.from_numpy(codes), torch.from_numpy(tiles).view(DTYPE[fmt]),
            None if rows is None else torch.from_numpy(rows).view(-1, 1))


def _values(q, blocks, scale):
    fmt = "nvfp4" if blocks.dtype == DTYPE["nvfp4"] else "mxfp4"
    v = f4.stored_values(q.numpy(), blocks.view(torch.uint8).numpy(), fmt)
    return v if scale is None else v * scale.double().numpy().reshape(-1, 1)


def _product(a, w, bias, gelu):
    y = _values(*a) @ _values(*w).T
    if bias is not None:
        y = y + bias.double().numpy()
    return torch.from_numpy(f4.gelu_tanh(y) if gelu else y).bfloat16()


def _install(dit):
    """The out-variant operators on CPU tensors, for this process."""
    fmt_of = lambda t: "nvfp4" if t.dtype == DTYPE["nvfp4"] else "mxfp4"  # noqa: E731

    def quant(q, blocks, scales, x, given):
        assert given is None
        for dst, src in zip((q, blocks.view(torch.uint8), scales),
                            (lambda c, b, s: (c, b.view(torch.uint8), s))(*_quant(x, fmt_of(blocks)))):
            if dst is not None:
                dst.copy_(src)

    def mm(out, a, b, blocks_a, blocks_b, scales_a, scales_b, bias, epilogue, tile, splits):
        assert tile == 0 and splits == 1
        out.copy_(_product((a, blocks_a, scales_a), (b.t().contiguous(), blocks_b, scales_b), bias,
                           epilogue == dit.ops.EPI_GELU_TANH))

    lib = torch.library.Library("taomate_w8a8", "IMPL", "CPU")
    lib.impl("scaled_fp4_quant", quant)
    lib.impl("scaled_mm_fp4", mm)
    dit.ops.scaled_fp4_quant = lambda x, *, block_format: _quant(x, block_format)
    return lib


def _weights(dit):
    cpu = torch.device("cpu")
    return (dit.random_bf16((FFN, D), 0.02, SEED + 10, cpu), dit.random_bf16((FFN,), 0.01, SEED + 11, cpu),
            dit.random_bf16((D, FFN), 0.02, SEED + 20, cpu))


def _worker(rank: int, world: int, port: int, out_dir: str, fmt: str) -> None:
    result = {"rank": rank, "ok": False}
    try:
        _init(rank, world, port)
        from taomate_hd_b200 import dit
        from taomate_hd_b200.parallel import ParallelContext

        lib = _install(dit)  # noqa: F841  kept while the operators run
        x = torch.randn(TOKENS, D, generator=torch.Generator().manual_seed(1)).bfloat16()
        w1, b1, w2 = _weights(dit)
        b2 = torch.full((D,), 3.0, dtype=torch.bfloat16)  # entering twice would show

        hidden = _product(_quant(x, fmt), _quant(w1, fmt), b1, True)
        partials = []
        for r in range(world):
            part = slice(r * FFN // world, (r + 1) * FFN // world)
            partials.append(_product(_quant(hidden[:, part].contiguous(), fmt),
                                     _quant(w2[:, part].contiguous(), fmt), b2 if r == 0 else None,
                                     False).float())
        want = sum(partials).bfloat16()
        ctx = ParallelContext(tp_world_size=world, tp_rank=rank,
                              tp_group=torch.distributed.group.WORLD)
        for reduce in ("reduce_scatter", "all_reduce"):
            mlp = dit.TPW4A4MLP(TOKENS, D, FFN, ctx, torch.device("cpu"), seed=SEED,
                                block_format=fmt, reduce=reduce)
            mlp.fc2.bias = b2
            rows = slice(rank * TOKENS // world, (rank + 1) * TOKENS // world)
            for _ in range(2):  # the buffers are reused
                got = mlp.forward(x)
                expect = want[rows] if reduce == "reduce_scatter" else want
                result[f"{reduce}_exact"] = bool(torch.equal(got, expect))
            local = hidden[:, rank * FFN // world:(rank + 1) * FFN // world]
            result[f"{reduce}_hidden"] = bool(torch.equal(mlp.h, local))
        full = torch.nn.functional.gelu(x.float() @ w1.float().t() + b1.float(), approximate="tanh")
        full = full @ w2.float().t() + 3.0
        result["far"] = float((want.float() - full).abs().max())
        for tokens, ffn in ((TOKENS, FFN + 2), (TOKENS, FFN + 32), (TOKENS + 1, FFN)):
            try:
                dit.TPW4A4MLP(tokens, D, ffn, ctx, torch.device("cpu"), block_format=fmt)
                result["refuses"] = False
            except ValueError:
                result.setdefault("refuses", True)
        result["ok"] = True
        torch.distributed.barrier()
        torch.distributed.destroy_process_group()
    except Exception:
        result["error"] = traceback.format_exc()
    Path(out_dir, f"rank{rank}.pkl").write_bytes(pickle.dumps(result))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_mlp_on_two_ranks(tmp_path, fmt):
    for res in _run(_worker, 2, tmp_path, fmt):
        assert res["ok"], res.get("error")
        assert res["reduce_scatter_hidden"] and res["all_reduce_hidden"]
        assert res["reduce_scatter_exact"] and res["all_reduce_exact"]
        assert res["refuses"]
        # 4 bits and bf16: an output of 3 + sum of 192 terms of about 0.1 x 0.02 each; a second
        # bias, or a missing one, would be off by 3
        assert res["far"] < 0.5


def test_row_scales_survive_column_sharding():
    """What the hidden columns' equality rests on: the codes and scales of a weight's rows
    do not depend on the other rows."""
    w = torch.randn(FFN, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    for fmt in DTYPE:
        q, b, s = _quant(w, fmt)
        qh, bh, sh = _quant(w[FFN // 2:], fmt)
        assert torch.equal(q[FFN // 2:], qh) and (s is None or torch.equal(s[FFN // 2:], sh))
        np.testing.assert_array_equal(_values(q, b, s)[FFN // 2:], _values(qh, bh, sh))
