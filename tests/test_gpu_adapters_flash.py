"""Adapters in a transformer whose middle blocks run on the rows that Flash selects."""
import pytest
import torch
from torch import nn

from helpers import bf16_randn
from lynnreal_omni_amd import adapters as L, flash
from test_flash_selection import _config, grid_layout
from test_gpu_adapters import make as some_adapters, spread

pytestmark = pytest.mark.gpu

WIDTH, COUNT = 64, 3


class Block(nn.Module):
    def __init__(self, seed):
        super().__init__()
        self.proj = nn.Linear(WIDTH, WIDTH)
        with torch.no_grad():
            g = torch.Generator().manual_seed(seed)
            self.proj.weight.copy_(torch.randn(WIDTH, WIDTH, generator=g) / 8)
            self.proj.bias.zero_()
        self.proj = self.proj.bfloat16().cuda()

    def forward(self, hidden, temb, indices, rotary, mask=None):
        return hidden + 0.1 * self.proj(hidden)


class Transformer(nn.Module):
    def __init__(self, fail_at=None):
        super().__init__()
        self.transformer_blocks = nn.ModuleList([Block(i) for i in range(8)])
        self.fail_at = fail_at

    def forward(self, hidden, temb, indices, rotary, position_ids, token_tags, mask=None):
        for i, block in enumerate(self.transformer_blocks):
            if i == self.fail_at:
                raise KeyError("stop")
            hidden = block(hidden, temb, indices, rotary, mask)
        return hidden


def inputs(batch):
    pos, tags = (t.cuda() for t in grid_layout(frames=3, height=10, width=14, text=11))
    n = tags.numel()
    g = torch.Generator().manual_seed(9)
    x = bf16_randn((batch, n, WIDTH), g).cuda()
    phase = torch.randn(n, 8, generator=g).cuda()
    picks = torch.tensor(spread(batch * n, COUNT)).view(batch, n)
    return x, (None, torch.randint(0, 6, (n,), generator=g).cuda(), (phase.cos(), phase.sin())), pos, tags, picks.cuda()


def adapters_of(names):
    return {name: L.LowRankAdapters(*some_adapters(COUNT, 8, WIDTH, WIDTH, torch.bfloat16, i)) for i, name in enumerate(names)}


@torch.inference_mode()
@pytest.mark.parametrize("first", ["flash", "adapters"])
@pytest.mark.parametrize("batch", [1, 2])
def test_adapters_follow_the_rows(batch, first):
    """Every block's tokens have their adapters, in the compressed blocks those of the rows that are kept."""
    x, rest, pos, tags, picks = inputs(batch)
    names = [f"transformer_blocks.{i}.proj" for i in (0, 2, 3, 5, 6)]
    model, beside = Transformer().eval(), adapters_of(names)
    config = _config(residual_gain=0.8)
    if first == "flash":
        flash.configure_flash(model, config)
    requests = L.adapt_transformer(model, beside)
    if first == "adapters":
        flash.configure_flash(model, config)
    none = model(x, *rest, pos, tags)
    plan = requests.plan = L.AdapterPlan(picks, COUNT)
    got = model(x, *rest, pos, tags)
    assert requests.plan is plan and torch.equal(model(x, *rest, pos, tags), got)

    keep, inverse = flash.spatial_layout(pos, tags)
    short = L.AdapterPlan(picks[:, keep].contiguous(), COUNT)
    blocks = Transformer().eval().transformer_blocks

    def run(hidden, span, plan):
        for i in span:
            y = blocks[i].proj(hidden)
            name = f"transformer_blocks.{i}.proj"
            hidden = hidden + 0.1 * (beside[name](hidden, y, plan) if name in beside else y)
        return hidden

    full = run(x, range(2), plan)
    small = full.index_select(1, keep)
    h = full + ((run(small, range(2, 6), short) - small) * 0.8).index_select(1, inverse)
    want = run(h, range(6, 8), plan)
    assert torch.equal(got, want) and not torch.equal(got, none)
    requests.plan = None
    assert torch.equal(model(x, *rest, pos, tags), none)


@torch.inference_mode()
def test_plans_of_their_own():
    """Requests of the compressed blocks alone, whose plan is over the kept rows, stay as they are."""
    x, rest, pos, tags, picks = inputs(1)
    outer, inner = (adapters_of([f"transformer_blocks.{i}.proj" for i in places]) for places in ((0, 7), (2, 4)))
    one, both = Transformer().eval(), Transformer().eval()
    for model in (one, both):
        flash.configure_flash(model, _config())
    requests = L.adapt_transformer(one, {**outer, **inner})
    requests.plan = L.AdapterPlan(picks, COUNT)
    keep, _ = flash.spatial_layout(pos, tags)
    a, b = L.adapt_transformer(both, outer), L.adapt_transformer(both, inner)
    a.plan, b.plan = requests.plan, L.AdapterPlan(picks[:, keep], COUNT)
    kept = b.plan
    assert torch.equal(both(x, *rest, pos, tags), one(x, *rest, pos, tags)) and b.plan is kept


@torch.inference_mode()
@pytest.mark.parametrize("fail_at", [3, 7])
def test_plan_after_an_error(fail_at):
    x, rest, pos, tags, picks = inputs(1)
    model = Transformer(fail_at).eval()
    flash.configure_flash(model, _config())
    requests = L.adapt_transformer(model, adapters_of(["transformer_blocks.2.proj", "transformer_blocks.3.proj"]))
    plan = requests.plan = L.AdapterPlan(picks, COUNT)
    with pytest.raises(KeyError):
        model(x, *rest, pos, tags)
    assert requests.plan is plan
    model.fail_at = None
    assert model(x, *rest, pos, tags).isfinite().all() and requests.plan is plan


@pytest.mark.parametrize("tokens,batch,count", [(1, 1, 1), (70, 1, 3), (300, 3, 40), (5000, 2, 1000)])
def test_rows_of_a_plan(tokens, batch, count):
    """The plan of some rows of each sequence, also after the plan has taken other indices."""
    g = torch.Generator().manual_seed(tokens)
    keep = (torch.rand(tokens, generator=g) < 0.4).nonzero()[:, 0]
    indices = [torch.randint(-2, count + 2, (batch, tokens), generator=g).cuda() for _ in range(2)]
    plan = L.AdapterPlan(indices[0], count)
    for given in indices:
        plan.update(given)
        got, want = plan.rows(keep.cuda(), batch), L.AdapterPlan(given[:, keep.cuda()], count)
        assert got.tokens == want.tokens == batch * len(keep) and got.adapters == count
        assert torch.equal(got.order, want.order) and torch.equal(got.tiles, want.tiles)
