"""The bench quotes the sort's DRAM traffic from the committed profile as long as that was taken from the sort's source as it is."""
import bench


def test_the_profile_is_of_the_source_that_is_built():
    call, one = bench.profiled_traffic()
    assert call and one and call > 4 * one  # a call is a histogram and four passes
