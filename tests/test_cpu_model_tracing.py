"""TinyGPT2 under torch.fx: a model that is called with tokens alone is traced as it was before it had losses, and the traced one has them too."""
import pytest
import torch

from nano_nccl_b200.models import TinyGPT2


def test_a_traced_model_has_logits_and_losses():
    torch.manual_seed(0)
    model = TinyGPT2(vocab=32, context=8, hidden=32, layers=1, heads=2)
    tokens, targets = torch.randint(0, 32, (2, 8)), torch.randint(-1, 32, (2, 8))
    traced = torch.fx.symbolic_trace(model)
    traced.graph.eliminate_dead_code()
    traced.recompile()
    assert torch.equal(traced(tokens), model(tokens))
    assert torch.equal(traced(tokens, targets), model(tokens, targets))
    with pytest.raises(ValueError, match="fused"):
        traced(tokens, teacher=(torch.ones(2, 8, 3), torch.zeros(2, 8, 3, dtype=torch.long)))
    with pytest.raises(ValueError, match="not both"):
        traced(tokens, targets, teacher=(1, 2))


def test_a_model_saved_before_it_had_losses():
    """Such a module, unpickled whole, has no choice of its vocabulary: it is the plain one."""
    torch.manual_seed(0)
    model = TinyGPT2(vocab=32, context=8, hidden=32, layers=1, heads=2)
    tokens, targets = torch.randint(0, 32, (2, 8)), torch.randint(-1, 32, (2, 8))
    want = model(tokens), model(tokens, targets)
    del model.vocabulary
    assert torch.equal(model(tokens), want[0]) and torch.equal(model(tokens, targets), want[1])
