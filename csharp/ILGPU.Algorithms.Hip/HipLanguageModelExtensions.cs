// Operators of language models beside the primitives: embedding lookup and its
// gradient, layer norm and its gradients, the norm of a list of gradients and its
// clipping.  The reference has no counterpart; names, argument order (stream, inputs,
// outputs, temp) and exception kinds follow its extension methods.  Views without a
// buffer (default) stand for what is optional.
using System;
using System.Collections.Generic;
using System.Runtime.InteropServices;
using ILGPU.Runtime;
using static ILGPU.Algorithms.Hip.HipAlgorithmsNativeMethods;

namespace ILGPU.Algorithms.Hip
{
    /// <summary>The upper half of a float, as raw bits.  The operators of this file take
    /// it; the primitives throw NotSupportedException.</summary>
    [StructLayout(LayoutKind.Sequential)]
    public struct HipBFloat16
    {
        public ushort Bits;
    }

    /// <summary>ilgpu_hip_tensor: one array of a list.</summary>
    [StructLayout(LayoutKind.Sequential)]
    internal unsafe struct HipTensor
    {
        public void* Data;
        public long Length;
        public int Type;
        public int Reserved;
    }

    /// <summary>Rows x columns elements of a view: element (r, c) is element
    /// r * RowStride + c of it.  A row stride of 0 (one row for all) is for matrices
    /// that are only read.</summary>
    public readonly struct HipMatrixView<T> where T : unmanaged
    {
        public HipMatrixView(ArrayView<T> view, long rows, long columns, long rowStride)
        {
            if (rows < 0 || columns < 0 || rowStride < 0 ||
                (rows > 0 && (columns > view.Length ||
                    (rowStride > 0 && rows - 1 > (view.Length - columns) / rowStride))))
                throw new ArgumentOutOfRangeException(nameof(view));
            View = view;
            Rows = rows;
            Columns = columns;
            RowStride = rowStride;
        }

        public HipMatrixView(ArrayView<T> view, long rows, long columns)
            : this(view, rows, columns, columns)
        { }

        public ArrayView<T> View { get; }
        public long Rows { get; }
        public long Columns { get; }
        public long RowStride { get; }

        internal unsafe void* Ptr => HipLanguageModelExtensions.PtrOf(View);
    }

    /// <summary>A list of views for the calls over many tensors.  It keeps their
    /// buffers: memory that nothing else refers to is not collected before the list
    /// is.</summary>
    public sealed unsafe class HipTensorList
    {
        private readonly List<HipTensor> tensors = new List<HipTensor>();
        private readonly List<object> views = new List<object>();

        public int Count => tensors.Count;

        public void Add<T>(ArrayView<T> view) where T : unmanaged
        {
            tensors.Add(new HipTensor
            {
                Data = HipLanguageModelExtensions.PtrOf(view),
                Length = view.Length,
                Type = HipTypeMap.ElementType<T>(),
            });
            views.Add(view);
        }

        internal HipTensor[] ToArray() => tensors.ToArray();
    }

    public static unsafe class HipLanguageModelExtensions
    {
        internal static void* PtrOf<T>(ArrayView<T> view) where T : unmanaged =>
            view.IsValid ? view.LoadEffectiveAddressAsPtr().ToPointer() : null;

        private static void CheckLength(bool fits, string name)
        {
            if (!fits)
                throw new ArgumentOutOfRangeException(name);
        }

        /// <summary>output[i] = scale * table[tokens[i]]; a token outside the table gives
        /// a row of zeros.</summary>
        public static void Embedding<T, TOutput, TToken>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<T> table,
            ArrayView<TToken> tokens,
            HipMatrixView<TOutput> output,
            float scale = 1.0f)
            where T : unmanaged
            where TOutput : unmanaged
            where TToken : unmanaged
        {
            CheckLength(
                output.Rows == tokens.Length && output.Columns == table.Columns,
                nameof(output));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_embedding(
                    HipStream.PtrOf(stream), table.Ptr, table.Rows, table.Columns,
                    table.RowStride, HipTypeMap.ElementType<T>(), PtrOf(tokens), tokens.Length,
                    HipTypeMap.ElementType<TToken>(), &scale, output.Ptr, output.RowStride,
                    HipTypeMap.ElementType<TOutput>()),
                nameof(table));
        }

        /// <summary>The temp of EmbeddingGradient in 32-bit integers.</summary>
        public static LongIndex1D ComputeEmbeddingGradientTempStorageSize(
            this HipAccelerator accelerator,
            LongIndex1D count,
            LongIndex1D vocabulary,
            LongIndex1D dimension)
        {
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_embedding_gradient_temp_bytes(
                    count, vocabulary, dimension, out long bytes),
                nameof(count));
            return HipTypeMap.BytesToInts(bytes);
        }

        /// <summary>gradTable[v] = scale * sum of gradOutput[i] over the positions i of
        /// token v; with accumulate added to what is there.</summary>
        public static void EmbeddingGradient<TGrad, T, TToken>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<TGrad> gradOutput,
            ArrayView<TToken> tokens,
            HipMatrixView<T> gradTable,
            ArrayView<int> temp,
            float scale = 1.0f,
            long paddingToken = -1,
            bool accumulate = false)
            where TGrad : unmanaged
            where T : unmanaged
            where TToken : unmanaged
        {
            CheckLength(gradOutput.Rows == tokens.Length, nameof(gradOutput));
            CheckLength(gradOutput.Columns == gradTable.Columns, nameof(gradTable));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_embedding_gradient(
                    HipStream.PtrOf(stream), gradOutput.Ptr, gradOutput.RowStride,
                    HipTypeMap.ElementType<TGrad>(), PtrOf(tokens), tokens.Length,
                    HipTypeMap.ElementType<TToken>(), &scale, paddingToken, accumulate ? 1 : 0,
                    gradTable.Ptr, gradTable.Rows, gradTable.Columns, gradTable.RowStride,
                    HipTypeMap.ElementType<T>(), PtrOf(temp), temp.Length * sizeof(int)),
                nameof(temp));
        }

        /// <summary>Layer norm of every row; mean and rstd are what the gradients need.
        /// </summary>
        public static void LayerNorm<T, TWeight>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<T> input,
            HipMatrixView<T> output,
            ArrayView<TWeight> weight,
            ArrayView<TWeight> bias,
            float epsilon,
            ArrayView<float> mean = default,
            ArrayView<float> rstd = default)
            where T : unmanaged
            where TWeight : unmanaged
        {
            CheckLength(
                output.Rows == input.Rows && output.Columns == input.Columns, nameof(output));
            CheckLength(!weight.IsValid || weight.Length == input.Columns, nameof(weight));
            CheckLength(!bias.IsValid || bias.Length == input.Columns, nameof(bias));
            CheckLength(!mean.IsValid || mean.Length >= input.Rows, nameof(mean));
            CheckLength(!rstd.IsValid || rstd.Length >= input.Rows, nameof(rstd));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_layer_norm(
                    HipStream.PtrOf(stream), input.Ptr, input.Rows, input.Columns,
                    input.RowStride, HipTypeMap.ElementType<T>(), PtrOf(weight), PtrOf(bias),
                    HipTypeMap.ElementType<TWeight>(), &epsilon, output.Ptr, output.RowStride,
                    (float*)PtrOf(mean), (float*)PtrOf(rstd)),
                nameof(input));
        }

        /// <summary>The temp of LayerNormGradient in 32-bit integers.</summary>
        public static LongIndex1D ComputeLayerNormGradientTempStorageSize(
            this HipAccelerator accelerator,
            LongIndex1D rows,
            LongIndex1D columns)
        {
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_layer_norm_gradient_temp_bytes(rows, columns, out long bytes),
                nameof(rows));
            return HipTypeMap.BytesToInts(bytes);
        }

        /// <summary>The gradients of LayerNorm; those given as default are not computed.
        /// With accumulate gradWeight and gradBias are added to.</summary>
        public static void LayerNormGradient<T, TWeight>(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipMatrixView<T> gradOutput,
            HipMatrixView<T> input,
            ArrayView<TWeight> weight,
            ArrayView<float> mean,
            ArrayView<float> rstd,
            HipMatrixView<T> gradInput,
            ArrayView<TWeight> gradWeight,
            ArrayView<TWeight> gradBias,
            ArrayView<int> temp,
            bool accumulate = false)
            where T : unmanaged
            where TWeight : unmanaged
        {
            CheckLength(
                gradOutput.Rows == input.Rows && gradOutput.Columns == input.Columns,
                nameof(gradOutput));
            CheckLength(
                !gradInput.View.IsValid ||
                (gradInput.Rows == input.Rows && gradInput.Columns == input.Columns),
                nameof(gradInput));
            CheckLength(!weight.IsValid || weight.Length == input.Columns, nameof(weight));
            CheckLength(
                !gradWeight.IsValid || gradWeight.Length == input.Columns, nameof(gradWeight));
            CheckLength(!gradBias.IsValid || gradBias.Length == input.Columns, nameof(gradBias));
            CheckLength(mean.Length >= input.Rows, nameof(mean));
            CheckLength(rstd.Length >= input.Rows, nameof(rstd));
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_layer_norm_gradient(
                    HipStream.PtrOf(stream), gradOutput.Ptr, gradOutput.RowStride, input.Ptr,
                    input.RowStride, input.Rows, input.Columns, HipTypeMap.ElementType<T>(),
                    PtrOf(weight), HipTypeMap.ElementType<TWeight>(), (float*)PtrOf(mean),
                    (float*)PtrOf(rstd), gradInput.Ptr, gradInput.RowStride, PtrOf(gradWeight),
                    PtrOf(gradBias), accumulate ? 1 : 0, PtrOf(temp),
                    temp.Length * sizeof(int)),
                nameof(temp));
        }

        /// <summary>The temp of GradientNorm in 32-bit integers.</summary>
        public static LongIndex1D ComputeGradientNormTempStorageSize(
            this HipAccelerator accelerator,
            LongIndex1D count)
        {
            HipAlgorithmsException.ThrowIfFailed(
                ilgpu_hip_gradient_norm_temp_bytes(count, out long bytes), nameof(count));
            return HipTypeMap.BytesToInts(bytes);
        }

        /// <summary>norm[0] = the root of the sum of the squares of all elements.</summary>
        public static void GradientNorm(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipTensorList gradients,
            ArrayView<float> norm,
            ArrayView<int> temp)
        {
            if (!norm.IsValid)
                throw new ArgumentNullException(nameof(norm));
            fixed (HipTensor* tensors = gradients.ToArray())
                HipAlgorithmsException.ThrowIfFailed(
                    ilgpu_hip_gradient_norm(
                        HipStream.PtrOf(stream), tensors, gradients.Count, (float*)PtrOf(norm),
                        PtrOf(temp), temp.Length * sizeof(int)),
                    nameof(temp));
            GC.KeepAlive(gradients);
        }

        /// <summary>gradients *= maxNorm / norm[0] where norm[0] is finite and the larger,
        /// in place or into targets.</summary>
        public static void ClipGradients(
            this HipAccelerator accelerator,
            AcceleratorStream stream,
            HipTensorList gradients,
            ArrayView<float> norm,
            float maxNorm,
            HipTensorList targets = null)
        {
            CheckLength(targets is null || targets.Count == gradients.Count, nameof(targets));
            if (!norm.IsValid)
                throw new ArgumentNullException(nameof(norm));
            fixed (HipTensor* sources = gradients.ToArray())
            fixed (HipTensor* places = targets?.ToArray())
                HipAlgorithmsException.ThrowIfFailed(
                    ilgpu_hip_clip_gradients(
                        HipStream.PtrOf(stream), sources, places, gradients.Count,
                        (float*)PtrOf(norm), &maxNorm),
                    nameof(gradients));
            GC.KeepAlive(gradients);
            GC.KeepAlive(targets);
        }
    }
}
