"""Which feed-forward blocks become gated pairs: those that compute ``down_proj(act_fn(gate_proj(x)) * up_proj(x))`` and nothing else."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

from bf16_huffman_infer_b200.functional import _activation_of, _is_gated_mlp


class Block(nn.Module):
    def __init__(self, act=None, hidden=64, inter=96, bias=False, **factory):
        super().__init__()
        factory = {"dtype": torch.bfloat16, **factory}
        self.gate_proj, self.up_proj = (nn.Linear(hidden, inter, bias=bias, **factory) for _ in range(2))
        self.down_proj = nn.Linear(inter, hidden, bias=bias, **factory)
        self.act_fn = act if act is not None else nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Clamped(Block):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x).clamp(max=7)) * self.up_proj(x).clamp(-7, 7))


class FarClamped(Block):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)).clamp(max=1e6) * self.up_proj(x))


class ClampedOutput(Block):
    def forward(self, x):
        return super().forward(x).clamp(-65504, 65504)


class Dropped(Block):
    def forward(self, x):
        return self.down_proj(F.dropout(self.act_fn(self.gate_proj(x)) * self.up_proj(x), 0.01, self.training))


class TrainingOnly(Block):
    def forward(self, x):
        return super().forward(x) * (1.5 if self.training else 1.0)


class Doubled(Block):
    def forward(self, x):
        return 2.0 * super().forward(x)


class Residual(Block):
    def forward(self, x):
        return x + super().forward(x)


class Scaled(Block):
    def forward(self, x):
        return super().forward(x * 0.5)


class Swapped(Block):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))


class Factor(Block):
    """A factor in a buffer, one as it is made and whatever a checkpoint brings."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.register_buffer("factor", torch.ones((), dtype=torch.bfloat16))

    def forward(self, x):
        return super().forward(x) * self.factor


class OneRowDiffers(Block):
    def forward(self, x):
        return super().forward(x) if x.numel() == x.size(-1) else super().forward(x).neg()


class NanToNum(Block):
    def forward(self, x):
        return self.down_proj((self.act_fn(self.gate_proj(x)) * self.up_proj(x)).nan_to_num())


class Around(Block):
    """Reads the weights itself, past whatever stands in the projections' places."""

    def forward(self, x):
        return self.down_proj(self.act_fn(F.linear(x, self.gate_proj.weight)) * self.up_proj(x))


class Pair(Block):
    def forward(self, x):
        return super().forward(x), None


class Written(Block):
    """The same, in other words."""

    def forward(self, hidden_states):
        up = self.up_proj(hidden_states)
        gate = self.gate_proj(hidden_states)
        return self.down_proj(self.act_fn(gate) * up)


class Chunked(Block):
    def forward(self, x):
        return torch.cat([Block.forward(self, part) for part in x.split(1, 0)])


class Clipped(nn.Module):
    def __init__(self, limit):
        super().__init__()
        self.limit = limit

    def forward(self, v):
        return F.silu(v).clamp(max=self.limit)


class Noisy(nn.Module):
    def forward(self, v):
        return F.silu(F.dropout(v, 1e-4, self.training))


def filled(block, value):
    for p in block.parameters():
        p.data.fill_(value)
    return block


@pytest.mark.parametrize("kind", [Clamped, FarClamped, ClampedOutput, Dropped, TrainingOnly, Doubled, Residual, Scaled, Swapped, Factor, OneRowDiffers, NanToNum, Around, Pair])
@pytest.mark.parametrize("weights", [None, 0.0, float("nan")])
@pytest.mark.parametrize("training", [False, True])
def test_blocks_that_do_something_else(kind, weights, training):
    """Whatever the weights are (a skeleton's zeros and NaNs agree with everything) and in either mode."""
    block = kind().train(training)
    assert _is_gated_mlp(block if weights is None else filled(block, weights)) is None


@pytest.mark.parametrize("act", [Clipped(7), Clipped(10), Clipped(1e20), Noisy(), nn.ReLU(), nn.PReLU(), nn.RReLU(), nn.Mish(), nn.LeakyReLU(), nn.Identity(),
                                 nn.Sequential(nn.SiLU(), nn.Dropout(0.01)), nn.GLU()])
def test_activations_that_are_something_else(act):
    for training in (False, True):
        act.train(training)
        assert _activation_of(act) is None and _is_gated_mlp(Block(act)) is None


@pytest.mark.parametrize("act,name", [("silu", "silu"), ("gelu", "gelu"), ("gelu_new", "gelu_tanh"), ("gelu_fast", "gelu_tanh"), ("gelu_pytorch_tanh", "gelu_tanh"),
                                      ("gelu_10", None), ("quick_gelu", None), ("relu2", None)])
def test_activations_by_their_library_names(act, name):
    from transformers.activations import ACT2FN
    assert _is_gated_mlp(Block(ACT2FN[act])) == name


def test_blocks_that_are_gated():
    for kind in (Block, Written, Chunked):
        for weights in (None, 0.0, float("nan")):
            for bias in (False, True):
                block = kind(bias=bias)
                block = block if weights is None else filled(block, weights)
                before = {k: v.clone() for k, v in block.state_dict().items()}
                modules, random = dict(block.named_modules()), torch.get_rng_state()
                assert _is_gated_mlp(block) == "silu"
                assert block.training and dict(block.named_modules()) == modules and torch.equal(torch.get_rng_state(), random)
                assert all(torch.equal(v.view(torch.int16), before[k].view(torch.int16)) for k, v in block.state_dict().items())
    for shape in ((32, 1), (32, 33), (160, 7), (64, 1000)):
        assert _is_gated_mlp(Block(None, *shape)) == "silu"


@pytest.mark.parametrize("module,name", [("qwen3", "Qwen3"), ("llama", "Llama"), ("mistral", "Mistral"), ("gemma", "Gemma")])
def test_blocks_of_the_library(module, name):
    import importlib
    lib = importlib.import_module(f"transformers.models.{module}.modeling_{module}")
    config = getattr(importlib.import_module(f"transformers.models.{module}.configuration_{module}"), name + "Config")(hidden_size=64, intermediate_size=96)
    block = getattr(lib, name + "MLP")(config).to(torch.bfloat16)
    assert _is_gated_mlp(block) == ("gelu_tanh" if module == "gemma" else "silu")


def test_somebodys_own_forward_stays():
    block = Block()
    block.gate_proj.forward = lambda x: nn.Linear.forward(block.gate_proj, x) * 2
    assert _is_gated_mlp(block) is None
