// Operators of recurrent language models beside those of HipLanguageModelExtensions: the
// gated recurrence with its gradients, the norms and the gate between two blocks with theirs,
// and the AdamW step.  The reference has no counterpart; names, argument order (stream,
// inputs, outputs, temp) and exception kinds follow its extension methods.  Views without a
// buffer (default) stand for what is optional.
using System;
using System.Runtime.InteropServices;
using ILGPU.Runtime;
using static ILGPU.Algorithms.Hip.HipAlgorithmsNativeMethods;

namespace ILGPU.Algorithms.Hip
{
    /// <summary>ilgpu_hip_decay.</summary>
    public enum HipDecayKind
    {
        Sigmoid = 0,
        Exponential = 1,
    }

    /// <summary>ilgpu_hip_gate.</summary>
    public enum HipGateKind
    {
        Sigmoid = 0,
        Silu = 1,
    }

    /// <summary>The sequences of a packed batch: equal parts of the rows, or cut at offsets
    /// (one more than sequences).</summary>
    public readonly struct HipPackedSequences<TOffset> where TOffset : unmanaged
    {
        public HipPackedSequences(long count, ArrayView<TOffset> offsets = default)
        {
            if (count < 0 || (offsets.IsValid && offsets.Length != count + 1))
                throw new ArgumentOutOfRangeException(nameof(offsets));
            Count = count;
            Offsets = offsets;
        }

        public long Count { get; }
        public ArrayView<TOffset> Offsets { get; }
    }

    /// <summary>What a block's output passes through on its way into the residual stream:
    /// a norm, a gate and a scale.  default passes it on as it is.</summary>
    public struct HipBlockOutput<T, TWeight>
        where T : unmanaged
        where TWeight : unmanaged
    {
        private float? scale;
        private HipGateKind? kind;

        public HipBlockOutput(float scale)
        {
            Normalized = false;
            Weight = default;
            Gate = default;
            kind = null;
            this.scale = scale;
        }

        public bool Normalized;
        public ArrayView<TWeight> Weight;
        public HipMatrixView<T> Gate;

        /// <summary>Silu where nothing was set.</summary>
        public HipGateKind Kind
        {
            get => kind ?? HipGateKind.Silu;
            set => kind = value;
        }

        /// <summary>1 where nothing was set.</summary>
        public float Scale
        {
            get => scale ?? 1.0f;
            set => scale = value;
        }
    }

    /// <summary>Where the gradients of ResidualNorm go; those left as default are not
    /// computed.</summary>
    public struct HipResidualNormGradients<T, TResidual, TWeight>
        where T : unmanaged
        where TResidual : unmanaged
        where TWeight : unmanaged
    {
        public HipMatrixView<T> Input;
        public HipMatrixView<T> Gate;
        public HipMatrixView<TResidual> Residual;
        public ArrayView<TWeight> InputWeight;
        public ArrayView<TWeight> Weight;
        public bool Accumulate;
    }

    /// <summary>ilgpu_hip_adamw_options.</summary>
    [StructLayout(LayoutKind.Sequential)]
    internal struct HipAdamWNumbers
    {
        public double Rate;
        public double Beta1;
        public double Beta2;
        public double Epsilon;
        public double WeightDecay;
        public double MaxNorm;
        public long Seed;
    }

    /// <summary>The numbers of an AdamW step.</summary>
    public sealed class HipAdamWOptions
    {
        public double Rate { get; set; } = 1e-3;
        public double Beta1 { get; set; } = 0.9;
        public double Beta2 { get; set; } = 0.999;
        public double Epsilon { get; set; } = 1e-8;
        public double WeightDecay { get; set; }
        public double MaxNorm { get; set; } = double.PositiveInfinity;
        public long Seed { get; set; }
    }

    /// <summary>A moment of AdamW: tensors of float, or of byte with a scale (float) for
    /// each 256 of their elements.</summary>
    public sealed class HipMoments
    {
        public HipMoments(HipTensorList values, HipTensorList scales = null)
        {
            Values = values;
            Scales = scales;
        }

        public HipTensorList Values { get; }
        public HipTensorList Scales { get; }
    }

    public static unsafe class HipRecurrentModelExtensions
    {
        private static void* PtrOf<T>(ArrayView<T> view) where T : unmanaged =>
            HipLanguageModelExtensions.PtrOf(view);

        private static void CheckLength(bool fits, string name)
        {
            if (!fits)
                throw new ArgumentOutOfRangeException(name);
        }

        private static bool SameShape<T>(HipMatrixView<T> view, long rows, long columns)
            where T : unmanaged =>
            !view.View.IsValid || (view.Rows == rows && view.Columns == columns);

        private static bool Fits<T>(ArrayView<T> view, long length) where T : unmanaged =>
            !view.IsValid || view.Length == length;

        /// <summary>The temp of GatedRecurrence and its gradient in 32-bit integers; 0 where
        /// so many rows need none.</summary>
        public static LongIndex1D ComputeGatedRecurrenceTempStorageSize(
            this HipAccelerator accelerator,
            LongIndex1D rows,
            LongIndex1D channels)
        {
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_gated_recurrence_temp_bytes(rows, channels, out long bytes),
                nameof(rows));
            return HipTypeMap.BytesToInts(bytes);
        }

        /// <summary>output[t] = h[t] = a * h[t-1] + b in every channel of every sequence, with
        /// a = sigmoid(gate) or exp(gate) and b = input or (1 - a) * input.</summary>
        public static void GatedRecurrence<T, TOffset>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<T> gate,
            HipMatrixView<T> input,
            HipMatrixView<T> output,
            HipPackedSequences<TOffset> sequences,
            HipDecayKind decay,
            bool complement,
            HipMatrixView<float> initial,
            HipMatrixView<float> final,
            ArrayView<int> temp)
            where T : unmanaged
            where TOffset : unmanaged
        {
            long rows = input.Rows, channels = input.Columns;
            CheckLength(gate.Rows == rows && gate.Columns == channels, nameof(gate));
            CheckLength(output.Rows == rows && output.Columns == channels, nameof(output));
            CheckLength(SameShape(initial, sequences.Count, channels), nameof(initial));
            CheckLength(SameShape(final, sequences.Count, channels), nameof(final));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_gated_recurrence(
                    HipStream.PtrOf(stream), gate.Ptr, gate.RowStride, input.Ptr,
                    input.RowStride, rows, channels, HipTypeMap.ElementType<T>(), (int)decay,
                    complement ? 1 : 0, PtrOf(sequences.Offsets),
                    HipTypeMap.ElementType<TOffset>(), sequences.Count, (float*)initial.Ptr,
                    initial.RowStride, output.Ptr, output.RowStride, (float*)final.Ptr,
                    final.RowStride, PtrOf(temp), temp.Length * sizeof(int)),
                nameof(temp));
        }

        /// <summary>The gradients of GatedRecurrence; those given as default are not computed.
        /// </summary>
        public static void GatedRecurrenceGradient<T, TOffset>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<T> gradOutput,
            HipMatrixView<T> gate,
            HipMatrixView<T> input,
            HipMatrixView<T> output,
            HipPackedSequences<TOffset> sequences,
            HipDecayKind decay,
            bool complement,
            HipMatrixView<float> initial,
            HipMatrixView<float> gradFinal,
            HipMatrixView<T> gradGate,
            HipMatrixView<T> gradInput,
            HipMatrixView<float> gradInitial,
            ArrayView<int> temp)
            where T : unmanaged
            where TOffset : unmanaged
        {
            long rows = input.Rows, channels = input.Columns;
            CheckLength(
                gradOutput.Rows == rows && gradOutput.Columns == channels, nameof(gradOutput));
            CheckLength(gate.Rows == rows && gate.Columns == channels, nameof(gate));
            CheckLength(output.Rows == rows && output.Columns == channels, nameof(output));
            CheckLength(SameShape(gradGate, rows, channels), nameof(gradGate));
            CheckLength(SameShape(gradInput, rows, channels), nameof(gradInput));
            CheckLength(SameShape(initial, sequences.Count, channels), nameof(initial));
            CheckLength(SameShape(gradFinal, sequences.Count, channels), nameof(gradFinal));
            CheckLength(SameShape(gradInitial, sequences.Count, channels), nameof(gradInitial));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_gated_recurrence_gradient(
                    HipStream.PtrOf(stream), gradOutput.Ptr, gradOutput.RowStride, gate.Ptr,
                    gate.RowStride, input.Ptr, input.RowStride, output.Ptr, output.RowStride,
                    rows, channels, HipTypeMap.ElementType<T>(), (int)decay, complement ? 1 : 0,
                    PtrOf(sequences.Offsets), HipTypeMap.ElementType<TOffset>(),
                    sequences.Count, (float*)initial.Ptr, initial.RowStride,
                    (float*)gradFinal.Ptr, gradFinal.RowStride, gradGate.Ptr,
                    gradGate.RowStride, gradInput.Ptr, gradInput.RowStride,
                    (float*)gradInitial.Ptr, gradInitial.RowStride, PtrOf(temp),
                    temp.Length * sizeof(int)),
                nameof(temp));
        }

        /// <summary>total = residual + scale * y and output = total * rstd * weight, with y the
        /// input behind its norm and gate.</summary>
        public static void ResidualNorm<T, TResidual, TWeight>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<T> input,
            HipBlockOutput<T, TWeight> block,
            HipMatrixView<TResidual> residual,
            HipMatrixView<TResidual> total,
            HipMatrixView<T> output,
            ArrayView<TWeight> weight,
            float epsilon,
            ArrayView<float> inputRstd = default,
            ArrayView<float> rstd = default)
            where T : unmanaged
            where TResidual : unmanaged
            where TWeight : unmanaged
        {
            long rows = input.Rows, columns = input.Columns;
            float scale = block.Scale;
            CheckLength(Fits(block.Weight, columns), nameof(block));
            CheckLength(SameShape(block.Gate, rows, columns), nameof(block));
            CheckLength(SameShape(residual, rows, columns), nameof(residual));
            CheckLength(SameShape(total, rows, columns), nameof(total));
            CheckLength(SameShape(output, rows, columns), nameof(output));
            CheckLength(Fits(weight, columns), nameof(weight));
            CheckLength(!inputRstd.IsValid || inputRstd.Length >= rows, nameof(inputRstd));
            CheckLength(!rstd.IsValid || rstd.Length >= rows, nameof(rstd));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_residual_norm(
                    HipStream.PtrOf(stream), input.Ptr, input.RowStride, rows, columns,
                    HipTypeMap.ElementType<T>(), block.Normalized ? 1 : 0, PtrOf(block.Weight),
                    block.Gate.Ptr, block.Gate.RowStride, (int)block.Kind, residual.Ptr,
                    residual.RowStride, HipTypeMap.ElementType<TResidual>(), &scale,
                    PtrOf(weight), HipTypeMap.ElementType<TWeight>(), &epsilon, total.Ptr,
                    total.RowStride, output.Ptr, output.RowStride, (float*)PtrOf(inputRstd),
                    (float*)PtrOf(rstd)),
                nameof(input));
        }

        /// <summary>The temp of ResidualNormGradient in 32-bit integers.</summary>
        public static LongIndex1D ComputeResidualNormGradientTempStorageSize(
            this HipAccelerator accelerator,
            LongIndex1D rows,
            LongIndex1D columns)
        {
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_residual_norm_gradient_temp_bytes(rows, columns, out long bytes),
                nameof(rows));
            return HipTypeMap.BytesToInts(bytes);
        }

        /// <summary>The gradients of ResidualNorm; gradOutput or gradTotal as default was not
        /// used.</summary>
        public static void ResidualNormGradient<T, TResidual, TWeight>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<T> gradOutput,
            HipMatrixView<TResidual> gradTotal,
            HipMatrixView<T> input,
            HipBlockOutput<T, TWeight> block,
            ArrayView<float> inputRstd,
            HipMatrixView<TResidual> total,
            ArrayView<TWeight> weight,
            ArrayView<float> rstd,
            HipResidualNormGradients<T, TResidual, TWeight> gradients,
            ArrayView<int> temp)
            where T : unmanaged
            where TResidual : unmanaged
            where TWeight : unmanaged
        {
            long rows = input.Rows, columns = input.Columns;
            float scale = block.Scale;
            CheckLength(SameShape(gradOutput, rows, columns), nameof(gradOutput));
            CheckLength(SameShape(gradTotal, rows, columns), nameof(gradTotal));
            CheckLength(SameShape(total, rows, columns), nameof(total));
            CheckLength(Fits(block.Weight, columns), nameof(block));
            CheckLength(SameShape(block.Gate, rows, columns), nameof(block));
            CheckLength(Fits(weight, columns), nameof(weight));
            CheckLength(!inputRstd.IsValid || inputRstd.Length >= rows, nameof(inputRstd));
            CheckLength(!rstd.IsValid || rstd.Length >= rows, nameof(rstd));
            CheckLength(
                SameShape(gradients.Input, rows, columns) &&
                SameShape(gradients.Gate, rows, columns) &&
                SameShape(gradients.Residual, rows, columns) &&
                Fits(gradients.InputWeight, columns) && Fits(gradients.Weight, columns),
                nameof(gradients));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_residual_norm_gradient(
                    HipStream.PtrOf(stream), gradOutput.Ptr, gradOutput.RowStride,
                    gradTotal.Ptr, gradTotal.RowStride, input.Ptr, input.RowStride, rows,
                    columns, HipTypeMap.ElementType<T>(), block.Normalized ? 1 : 0,
                    PtrOf(block.Weight), (float*)PtrOf(inputRstd), block.Gate.Ptr,
                    block.Gate.RowStride, (int)block.Kind, total.Ptr, total.RowStride,
                    HipTypeMap.ElementType<TResidual>(), &scale, PtrOf(weight),
                    HipTypeMap.ElementType<TWeight>(), (float*)PtrOf(rstd),
                    gradients.Input.Ptr, gradients.Input.RowStride, gradients.Gate.Ptr,
                    gradients.Gate.RowStride, gradients.Residual.Ptr,
                    gradients.Residual.RowStride, PtrOf(gradients.InputWeight),
                    PtrOf(gradients.Weight), gradients.Accumulate ? 1 : 0, PtrOf(temp),
                    temp.Length * sizeof(int)),
                nameof(temp));
        }

        /// <summary>One step of AdamW, in place.  step counts on the device, 1 for the first;
        /// schedule and norm are on the device too.</summary>
        public static void AdamW(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipTensorList parameters,
            HipTensorList gradients,
            HipMoments first,
            HipMoments second,
            HipAdamWOptions options,
            ArrayView<long> step,
            HipTensorList copies = null,
            ArrayView<float> schedule = default,
            ArrayView<float> norm = default)
        {
            int count = parameters.Count;
            CheckLength(gradients.Count == count, nameof(gradients));
            CheckLength(
                first.Values.Count == count && (first.Scales?.Count ?? count) == count,
                nameof(first));
            CheckLength(
                second.Values.Count == count && (second.Scales?.Count ?? count) == count,
                nameof(second));
            CheckLength((copies?.Count ?? count) == count, nameof(copies));
            if (!step.IsValid)
                throw new ArgumentNullException(nameof(step));
            var numbers = new HipAdamWNumbers
            {
                Rate = options.Rate,
                Beta1 = options.Beta1,
                Beta2 = options.Beta2,
                Epsilon = options.Epsilon,
                WeightDecay = options.WeightDecay,
                MaxNorm = options.MaxNorm,
                Seed = options.Seed,
            };
            fixed (HipTensor* p = parameters.ToArray())
            fixed (HipTensor* g = gradients.ToArray())
            fixed (HipTensor* m = first.Values.ToArray())
            fixed (HipTensor* v = second.Values.ToArray())
            fixed (HipTensor* ms = first.Scales?.ToArray())
            fixed (HipTensor* vs = second.Scales?.ToArray())
            fixed (HipTensor* c = copies?.ToArray())
                HipAlgorithmsException.ThrowIfFailed(
                    ilgpu_hip_adamw(
                        HipStream.PtrOf(stream), p, g, m, v, ms, vs, c, count, &numbers,
                        (long*)PtrOf(step), (float*)PtrOf(schedule), (float*)PtrOf(norm)),
                    nameof(parameters));
            GC.KeepAlive(parameters);
            GC.KeepAlive(gradients);
            GC.KeepAlive(first);
            GC.KeepAlive(second);
            GC.KeepAlive(copies);
        }

        /// <summary>8-bit moments as the numbers they stand for.</summary>
        public static void AdamWMoments(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMoments first,
            HipTensorList firstTargets,
            HipMoments second,
            HipTensorList secondTargets)
        {
            int count = firstTargets.Count;
            CheckLength(
                first.Values.Count == count && first.Scales?.Count == count, nameof(first));
            CheckLength(
                second.Values.Count == count && second.Scales?.Count == count, nameof(second));
            CheckLength(secondTargets.Count == count, nameof(secondTargets));
            fixed (HipTensor* m = first.Values.ToArray())
            fixed (HipTensor* ms = first.Scales.ToArray())
            fixed (HipTensor* mt = firstTargets.ToArray())
            fixed (HipTensor* v = second.Values.ToArray())
            fixed (HipTensor* vs = second.Scales.ToArray())
            fixed (HipTensor* vt = secondTargets.ToArray())
                HipAlgorithmsException.ThrowIfFailed(
                    ilgpu_hip_adamw_moments(
                        HipStream.PtrOf(stream), m, ms, mt, v, vs, vt, count),
                    nameof(first));
            GC.KeepAlive(first);
            GC.KeepAlive(firstTargets);
            GC.KeepAlive(second);
            GC.KeepAlive(secondTargets);
        }
    }
}
