"""Rotation of rows of negative positions on the GPU: what a new tensor holds there, and what TKM_ROPE_CLEAR writes."""
import pytest
import torch

from kv_cases import DT

pytestmark = pytest.mark.gpu


def nan_everywhere(shape, dtype, dev):
    """Leaves freed memory of NaN where a new tensor of this size is likely to come from."""
    for _ in range(4):
        torch.full(shape, float("nan"), dtype=dtype, device=dev)


@pytest.mark.parametrize("rows,Hq,Hkv,D,rot", [(1, 1, 0, 64, 64), (7, 4, 2, 128, 96), (300, 3, 1, 64, 20), (4200, 2, 1, 128, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_new_tensors_hold_zeros(gpu, rows, Hq, Hkv, D, rot, dtype, layout):
    """A padded batch's gradient has 0 in its padding, all heads of it; other rows are those of a given tensor."""
    from tokamak_amd import attn
    print(f"[case] rows {rows} Hq{Hq} Hkv{Hkv} D{D} rot {rot} {dtype} {layout}", flush=True)
    g, W = torch.Generator().manual_seed(rows), (Hq + 2 * Hkv) * D
    x = torch.randn(rows, W, generator=g).to(DT[dtype]).to(gpu)
    pos = torch.randint(-2, 4, (rows,), generator=g).to(torch.int32)
    pos[0] = -1
    rope, gone = attn.Rope(rot, layout=layout), (pos < 0).to(gpu)
    for call in (attn.rope_fwd, attn.rope_bwd):
        given = torch.full_like(x, 3.0)
        call(x, rope, Hq, Hkv, D, pos.to(gpu), None, given)
        assert (given[gone] == 3.0).all()
        nan_everywhere(x.shape, x.dtype, gpu)
        new = call(x, rope, Hq, Hkv, D, pos.to(gpu))
        assert attn.last_kernels() == ["rope"]
        assert (new[gone] == 0.0).all() and torch.equal(new[~gone], given[~gone])


def test_clear_of_given_rows(gpu):
    """The C call's flag, on rows further apart and in place; what lies between the rows stays."""
    from tokamak_amd import attn
    L, rope, W = attn.lib(), attn.Rope(64), 4 * 64
    x = torch.randn(5, W + 8, generator=torch.Generator().manual_seed(1)).half().to(gpu)
    pos = torch.tensor([3, -1, 0, -7, 2], dtype=torch.int32, device=gpu)
    for inverse in (0, 1):
        want = torch.zeros(5, W, dtype=torch.float16, device=gpu)
        (attn.rope_bwd if inverse else attn.rope_fwd)(x[:, :W], rope, 2, 1, 64, pos, None, want)
        for out in (torch.full_like(x, 5.0), x.clone()):
            src, rest = (x, 5.0) if out[0, W] == 5.0 else (out, x[:, W:].clone())
            assert L.tkm_attn_rope_rows(rope._ref, src.data_ptr(), W + 8, out.data_ptr(), W + 8, pos.data_ptr(), 1, 5, 2, 1, 64, 0,
                                        inverse | attn.ROPE_CLEAR, torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(out[:, :W], want) and (out[:, W:] == rest).all()
