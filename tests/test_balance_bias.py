"""The balance bias of a router stays fp32 whatever the module is cast to."""
import pytest
import torch


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16),
                                  lambda m: torch.nn.ModuleList([m]).bfloat16()[0]])
def test_casts_leave_it_in_fp32(cast):
    import memory_b200 as M
    r = M.ChapterRouter(8, 6, top_k=2, balance_bias=True)
    r.balance_bias.copy_(torch.linspace(-0.31, 0.4, 6))
    before = r.balance_bias.clone()
    got = cast(r)
    assert got.balance_bias.dtype == torch.float32 and torch.equal(got.balance_bias, before)
    assert got.router.weight.dtype != torch.float32 and "balance_bias" in got.state_dict()
    assert got.float().balance_bias.dtype == torch.float32
    assert M.ChapterRouter(8, 6).bfloat16().balance_bias is None


def test_it_moves_with_the_module():
    import memory_b200 as M
    r = M.ChapterRouter(8, 6, top_k=2, balance_bias=True)
    assert r.to(device="meta", dtype=torch.bfloat16).balance_bias.is_meta and r.balance_bias.dtype == torch.float32
    assert r.to_empty(device="cpu").balance_bias.device.type == "cpu"


@pytest.mark.gpu
def test_a_bf16_router_balances():
    import memory_b200 as M
    torch.manual_seed(0)
    r = M.ChapterRouter(64, 17, top_k=2, score="sigmoid", balance_bias=True).cuda().bfloat16()
    assert r.balance_bias.is_cuda
    r.balance_bias.fill_(0.5)
    r.route_token_level(torch.randn(1, 200, 64, device="cuda").bfloat16())
    load = r.last_load.clone()
    for _ in range(3):
        r.update_balance(0.001, load=load)
    sign = torch.sign(load.double().mean() - load).cpu()
    # three fp32 additions to numbers around 0.5, half a step of 2^-24 each
    assert ((r.balance_bias.double().cpu() - 0.5 - 0.003 * sign).abs() <= 3 * 2.0 ** -24 + 0.003 * 2.0 ** -24).all()
