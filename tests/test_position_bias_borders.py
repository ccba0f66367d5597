"""The bucket borders are made of plain whole numbers, whoever asks for them."""
import pytest
import torch


def test_borders_of_a_traced_size_are_whole_numbers():
    """A tracer's sizes are tensors: none may end up among the borders, or as the key of what is kept."""
    from torchgt_b200.position_bias import bucket_borders
    seen = []

    def borders_of(table):
        seen.append(bucket_borders(table.shape[0], 300, True))
        return table * 1
    for _ in range(2):
        torch.jit.trace(borders_of, (torch.zeros(38, 2),), check_trace=False)
    want = bucket_borders(38, 300, True)
    assert all(b is want for b in seen) and all(type(b) is int for b in want)


@pytest.mark.parametrize("buckets,distance", [(32.0, 128), (32, 128.0), (32, 100.5)])
def test_sizes_that_are_no_whole_numbers_are_refused(buckets, distance):
    from torchgt_b200 import RelativePositionBias
    from torchgt_b200.position_bias import bucket_borders
    bucket_borders(32, 128, True)                            # and stay refused where the same size is known
    with pytest.raises(TypeError):
        bucket_borders(buckets, distance, True)
    with pytest.raises(TypeError):
        RelativePositionBias(8, buckets, distance)
