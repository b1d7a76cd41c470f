"""Microscaled matrices without a GPU: shapes, refusals, the option's way through the model and the command line, which kernel a product takes."""
import pytest
import torch

from minfer_amd.cli import main, parse_args
from minfer_amd.kernels import ops
from test_registers import _scratch_bytes
from tiny import TINY_A


def test_shapes():
    assert ops.mx4_shapes(1, 1) == ((1, 1, 64, 16), (1, 1, 64, 4))
    assert ops.mx4_shapes(16, 512) == ((1, 4, 64, 16), (1, 1, 64, 4))
    assert ops.mx4_shapes(17, 513) == ((2, 5, 64, 16), (2, 2, 64, 4))
    codes, powers = ops.mx4_shapes(37888, 3584)
    assert torch.Size(codes).numel() + torch.Size(powers).numel() == 37888 * 3584 * 17 // 32


def test_pairs():
    gate, up = torch.arange(2 * 3 * 64 * 16, dtype=torch.int32).view(2, 3, 64, 16).to(torch.uint8), torch.zeros((2, 3, 64, 16), dtype=torch.uint8)
    both = ops.mx4_pairs(gate, up)
    assert both.shape == (4, 3, 64, 16) and torch.equal(both[0], gate[0]) and torch.equal(both[2], gate[1]) and not both[1::2].any()
    stacked = ops.mx4_pairs(gate[None].expand(5, -1, -1, -1, -1), up[None].expand(5, -1, -1, -1, -1))
    assert stacked.shape == (5, 4, 3, 64, 16) and torch.equal(stacked[3], both)
    with pytest.raises(ops.KernelError):
        ops.mx4_pairs(gate, up[:1])


def test_host_tensors_are_refused():
    codes, powers = (torch.zeros(s, dtype=torch.uint8) for s in ops.mx4_shapes(32, 64))
    x, out = torch.zeros((3, 64)), torch.zeros((3, 32))
    for call in (lambda: ops.mx4_quantise(torch.zeros((32, 64)), codes, powers), lambda: ops.mx4_dequantise(codes, powers, torch.zeros((32, 64))),
                 lambda: ops.mx4_linear(x, codes, powers, None, out), lambda: ops.mx4_linear_swiglu(x, codes, powers, out.to(torch.bfloat16)),
                 lambda: ops.mx4_moe_sparse(x, codes[None], powers[None], codes[None], powers[None], torch.zeros((3, 1), dtype=torch.int32),
                                            torch.ones((3, 1)), x, 32)):
        with pytest.raises(ops.KernelError, match="GPU"):
            call()


@pytest.mark.parametrize("m", [1, 16, 17, 64, 65, 128, 300, 2048, 4096, 16384])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (896, 896), (3584, 18944), (4608, 3584), (152064, 3584), (100, 40000)])
def test_every_plan_covers_its_product(m, n, k):
    """The parts of K of a plan cover it, none of them is empty, and the scratch is that of its kernels."""
    for epi, whole in ((ops.EPI_F32, 1), (ops.EPI_F32, 2), (ops.EPI_SWIGLU, 1), (ops.EPI_SWIGLU, 2), (ops.EPI_BF16, 0), (ops.EPI_SWIGLU, 0)):
        form, splits, six, parts = ops._mx4_plan(m, n, k, epi, whole, 256)
        groups, steps, w16 = -(-k // 512), -(-k // 128), -(-n // 16) * (2 if epi == ops.EPI_SWIGLU else 1)
        per = -(-groups // splits)
        assert 1 <= splits <= groups and (splits - 1) * per < groups <= splits * per
        assert parts == (splits * m * w16 * 16 if splits > 1 else 0)
        assert m <= 16 and whole or form > 0
        assert six == (0 if form == 0 else -(-m // 32) * (steps * 3 * 1024 + groups * 512))


def test_sizes_that_no_product_takes():
    for m, n, k in ((1, 16, (1 << 23) + 1), (1 << 30, 16, 1 << 20), (1, (1 << 30) + 1, 16)):
        with pytest.raises(ops.KernelError, match="mx4_linear"):
            ops._mx4_plan(m, n, k, ops.EPI_F32, 1, 256)


@pytest.mark.parametrize("limit", [-1.0, float("nan")])
def test_a_limit_that_is_none(limit, monkeypatch):
    monkeypatch.setattr(ops, "_need", lambda *a: None)
    codes, powers = (torch.zeros(s, dtype=torch.uint8) for s in ops._mx4_pair_shapes(32, 64))
    with pytest.raises(ops.KernelError, match="limit"):
        ops.mx4_linear_swiglu(torch.zeros((3, 64)), codes, powers, torch.zeros((3, 32), dtype=torch.bfloat16), limit=limit)


def test_streams_of_matrices_spill_nothing(tmp_path):
    """As in the products of bfloat16 matrices: a reload would wait for the weights in flight."""
    from minfer_amd.kernels import build
    for name, kinds in (("gemm_mx4", ("few_kernel", "few_six_kernel", "rows_kernel")), ("moe_mx4", ("experts_up_kernel", "experts_down_kernel")),
                        ("mx4", ("mx4_quantise_kernel", "mx4_dequantise_kernel"))):
        if not build.is_current(name):
            build.compile_library(name)
        scratch = _scratch_bytes(build.lib_path(name), str(tmp_path))
        assert all(any(k + "I" in n for n in scratch) for k in kinds)
        assert not {n: b for n, b in scratch.items() if b and any(k + "I" in n for k in kinds)}


def test_weights_option():
    from minfer_amd import config_from_dict
    from minfer_amd.engine.model import DecoderModel
    spec = config_from_dict(TINY_A).model_spec()
    model = DecoderModel(spec, torch.bfloat16, "cpu", "mx4")
    assert model.rt.mx4 and model.expected_tensors() == DecoderModel(spec, torch.bfloat16, "cpu").expected_tensors()
    with pytest.raises(ValueError, match="bfloat16"):
        DecoderModel(spec, torch.float32, "cpu", "mx4")
    with pytest.raises(ValueError, match="int3"):
        DecoderModel(spec, torch.bfloat16, "cpu", "int3")


def test_command_line(capsys):
    assert parse_args(["m", "--prompt-tokens", "1"])["weights"] == "stored"
    assert parse_args(["m", "--prompt-tokens", "1", "--weights", "mx4"])["weights"] == "mx4"
    assert main(["m", "--prompt-tokens", "1", "--weights", "int3"]) == 1 and "--weights" in capsys.readouterr().err
    assert main(["m", "--prompt-tokens", "1", "--weights", "mx4", "--dtype", "float32"]) == 1 and "bfloat16" in capsys.readouterr().err
