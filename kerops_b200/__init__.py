"""kerops_b200 - depthwise 3x3x3 channels-last fp16 convolution (forward and weight gradient)
for NVIDIA B200, behind the call signatures of kerops.ops.conv.DWConv / DWConvWGRAD, and the channel-mixing products that
follow it (ops.linear): grouped by expert with their gradients, and in 8-bit integers."""
__version__ = '0.1.0'
