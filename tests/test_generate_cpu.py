"""LinearAttnLM.generate's handling of lengths, with the model's two calls stood in
for (they need a GPU): the logits name the token read and its place."""
import pytest
import torch

from mamba_amd.models.linear_attn_lm import LinearAttnLM, LinearAttnLMConfig


class Echo(LinearAttnLM):
    """Answers with the row's last token of the prompt, then one more each step."""

    def forward(self, input_ids, lengths=None, states=None):
        n = torch.full((len(input_ids),), input_ids.shape[1]) if lengths is None else lengths.clamp(0, input_ids.shape[1])
        live = torch.arange(input_ids.shape[1])[None] < n[:, None]
        return torch.nn.functional.one_hot(torch.where(live, input_ids, 0), 50).float()

    def step(self, input_ids, states):
        return torch.nn.functional.one_hot(input_ids + 1, 50).float()


@pytest.fixture
def model():
    return Echo(LinearAttnLMConfig(vocab_size=50, model_dim=16, num_layers=1, head_dim=16))


IDS = torch.tensor([[5, 6, 7, 8], [10, 11, 12, 13], [20, 21, 22, 23]])


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_lengths(model, dtype):
    assert model.generate(IDS, 3).tolist() == [[8, 9, 10], [13, 14, 15], [23, 24, 25]]
    n = torch.tensor([4, 1, 3], dtype=dtype)
    assert model.generate(IDS, 2, lengths=n).tolist() == [[8, 9], [10, 11], [22, 23]]
    # a length past the row is the row's, as in the operator
    assert model.generate(IDS, 2, lengths=torch.tensor([5, 1000, 2], dtype=dtype)).tolist() == [[8, 9], [13, 14], [21, 22]]


def test_nothing_to_answer(model):
    for n in (0, -1):
        got = model.generate(IDS, n)
        assert got.shape == (3, 0) and got.dtype == IDS.dtype


def test_rows_without_a_token_are_refused(model):
    for n in ([4, 0, 3], [4, -2, 3]):
        with pytest.raises(ValueError, match="nothing to continue"):
            model.generate(IDS, 2, lengths=torch.tensor(n))
    with pytest.raises(ValueError, match="nothing to continue"):
        model.generate(IDS[:, :0], 2)
    with pytest.raises(ValueError, match="lengths has shape"):
        model.generate(IDS, 2, lengths=torch.tensor([3]))
