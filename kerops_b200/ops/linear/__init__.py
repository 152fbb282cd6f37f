from .grouped_linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD
from .int8_linear import Int8Linear, QuantRows

__all__ = ['GroupedLinear', 'GroupedLinearDGRAD', 'GroupedLinearWGRAD', 'Int8Linear', 'QuantRows']
